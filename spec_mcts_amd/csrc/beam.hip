// Beam search: the best continuations of each group of beams, and the states that follow them.
//
// Selection.  Candidate (beam r, token t) of a group has the score  scores[r] + x[r][t] - log sum_t' exp(x[r][t']);  the n best leave in descending order,
// equal ones by (beam, token).  A first launch goes over each row once, a workgroup per slice of it: the slice's values stay in registers while its maximum, its sum of
// exponentials and its n largest values are found.  A second one has a wave per group: it adds the slices' sums up and merges their sorted lists.
//   Order: within a row the fp16 values order exactly; between rows the scores are compared in 64 bits, with sums whose terms are fp32 (2^-23 each, the sum of a
//   slice in 64 bits), so that candidates keep their order unless they are closer than that.
// Bound: HBM, 2 bytes a logit; the smallest calls by the two launches.
//
// Reordering.  Row i of a group takes the contents of row parents[i], in place: a workgroup owns a strip of all rows of a group, has it in LDS and then writes.
// Bound: HBM, each row that moves read and written once.
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
    uint32_t b = __builtin_bit_cast(uint16_t, x);
    if ((b & 0x7FFFu) > 0x7C00u) b = 0xFC00u;      // NaN: -infinity
    if (b == 0x8000u) b = 0;                       // -0 is 0
    return b & 0x8000u ? 0xFFFFu - b : b | 0x8000u;
}
__device__ __forceinline__ float beam_value(uint32_t order) {
    const uint32_t b = order & 0x8000u ? order & 0x7FFFu : 0xFFFFu - order;
    return fminf((float)__builtin_bit_cast(half_t, (uint16_t)b), 65536.0f);      // (an infinity is the step after 65504: the others of its row stay in order)
}
__device__ __forceinline__ uint32_t beam_key(half_t x, int col) { return beam_order(x) << 16 | (0xFFFFu - (uint32_t)col); }

// exp(x), x <= 0, with the rounding of x log2(e) made good: about 2^-23
__device__ __forceinline__ float beam_exp(float x) {
    if (x < -104.0f) return 0.0f;                  // (below the least float; x may be -infinity)
    const float hi = x * 1.44269504f, lo = __builtin_fmaf(x, 1.44269504f, -hi) + x * 1.92596299e-8f;
    const float e = __builtin_amdgcn_exp2f(hi);
    return __builtin_fmaf(e * 0.693147181f, lo, e);
}

// 256 threads, VPT values each: a slice of 256 * VPT columns.
template <int VPT>
__global__ __launch_bounds__(256) void beam_slice_kernel(SelectParams p) {
    constexpr int CHUNKS = VPT / 8;
    __shared__ uint32_t top[256];                  // each thread's largest key
    __shared__ uint32_t found[VPT * BEAM_MAX_N];   // keys not below the n-th of them: at most VPT of each of n threads
    __shared__ uint32_t red_max[4];
    __shared__ double red_sum[4];
    __shared__ int n_found;
    const int slice = blockIdx.x, row = blockIdx.y, t = threadIdx.x, lane = t & 63, wave = t >> 6;
    const int c0 = slice * p.width, cols = min(p.width, p.vocab - c0), n = p.n;
    uint32_t *cand = p.cand + ((long)row * p.slices + slice) * n;
    const float score = p.scores[row];
    const bool ended = p.ended != nullptr && p.ended[row] != 0, lost = !(score > -INFINITY);
    if (ended || lost) {
        // No value counts: a lost beam's candidates are all -infinity and go by their index; of an ended beam's the first is its end, the others go by index
        // too (which the second launch does, too)
        return;
    }
    const half_t *x = p.logits + (long)row * p.ld + c0;
    uint32_t key[VPT];
    uint32_t mine = 0;
    const bool aligned = ((uintptr_t)x & 15) == 0;
#pragma unroll
    for (int i = 0; i < CHUNKS; ++i) {
        const int col = (i * 256 + t) * 8;
        h8 v;
        if (aligned && col + 8 <= cols) v = *reinterpret_cast<const h8 *>(x + col);
        else {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = col + e < cols ? x[col + e] : (half_t)0.0f;
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            key[i * 8 + e] = col + e < cols ? beam_key(v[e], col + e) : 0u;
            mine = max(mine, key[i * 8 + e]);
        }
    }
    top[t] = mine;
    uint32_t most = mine;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) most = max(most, (uint32_t)__shfl_xor((int)most, o, 64));
    if (lane == 0) red_max[wave] = most;
    if (t == 0) n_found = 0;
    __syncthreads();
    const float m = beam_value(max(max(red_max[0], red_max[1]), max(red_max[2], red_max[3])) >> 16);      // (every slice has a column)
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < VPT; ++i)
        if (key[i] != 0) {
            const float v = beam_value(key[i] >> 16);
            sum += v == m ? 1.0f : beam_exp(v - m);                    // (v == m: also both -infinity)
        }
    double total = sum;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) total += __shfl_xor(total, o, 64);
    if (lane == 0) red_sum[wave] = total;
    // the n-th largest of the threads' largest keys, bit by bit: n keys are not below it, and no key below it is among the n largest
    uint32_t mx[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) mx[i] = top[i * 64 + lane];
    uint32_t bar = 0;
#pragma unroll
    for (int bit = 31; bit >= 0; --bit) {
        const uint32_t at = bar | 1u << bit;
        int c = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) c += __popcll(__ballot(mx[i] >= at));
        if (c >= n) bar = at;
    }
#pragma unroll
    for (int i = 0; i < VPT; ++i)
        if (key[i] >= bar && key[i] != 0) found[atomicAdd(&n_found, 1)] = key[i];
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

// A wave per group.  Lane l has the lists l, l + 64, ..: list = row of the group * slices + slice.
__global__ __launch_bounds__(64) void beam_merge_kernel(SelectParams p) {
    extern __shared__ int at[];                    // [lists]: entries taken; then the rows' maxima and log sums
    const int g = blockIdx.x, lane = threadIdx.x, lists = p.W * p.slices;
    double *base = reinterpret_cast<double *>(at + ((lists + 1) & ~1));      // [W]: score - max - log sum
    float *row_max = reinterpret_cast<float *>(base + p.W);                   // [W]
    for (int i = lane; i < lists; i += 64) at[i] = 0;
    for (int r = lane; r < p.W; r += 64) {
        const long row = (long)g * p.W + r;
        const float score = p.scores[row];
        const bool ended = p.ended != nullptr && p.ended[row] != 0;
        float m = -INFINITY;
        double s = 0.0;
        if (score > -INFINITY && !ended) {
            for (int i = 0; i < p.slices; ++i) m = fmaxf(m, p.slice_max[row * p.slices + i]);
            for (int i = 0; i < p.slices; ++i) {
                const float mi = p.slice_max[row * p.slices + i];
                s += p.slice_sum[row * p.slices + i] * (mi == m ? 1.0 : exp((double)mi - (double)m));
            }
        }
        base[r] = (double)score - log(s);
        row_max[r] = m;
    }
    __syncthreads();
    auto head = [&](int list, double &value, long &index) {            // the list's next candidate
        const int r = list / p.slices, slice = list - r * p.slices, i = at[list];
        const long row = (long)g * p.W + r;
        const float score = p.scores[row];
        const bool ended = p.ended != nullptr && p.ended[row] != 0;
        value = -INFINITY;
        index = LONG_MAX;
        if (!(score > -INFINITY) || ended) {       // one list stands for the whole row
            if (slice != 0 || i >= p.vocab) return;
            int token = i;
            if (ended && score > -INFINITY) {
                token = i == 0 ? p.eos : i - 1 < p.eos ? i - 1 : i;
                if (i == 0) value = score;
            }
            index = (long)r * p.vocab + token;
            return;
        }
        const uint32_t key = i < p.n ? p.cand[(row * p.slices + slice) * p.n + i] : 0u;
        if (key == 0) return;
        index = (long)r * p.vocab + slice * p.width + (0xFFFFu - (key & 0xFFFFu));
        const float v = beam_value(key >> 16), m = row_max[r];
        value = v == -INFINITY ? -INFINITY : base[r] + (v == m ? 0.0 : (double)v - (double)m);
    };
    auto better = [](double v, long i, double w, long j) { return v > w || (v == w && i < j); };
    double best = -INFINITY;
    long index = LONG_MAX;
    int list = -1;
    auto mine = [&]() {                            // the best of the lane's lists
        best = -INFINITY;
        index = LONG_MAX;
        list = -1;
        for (int i = lane; i < lists; i += 64) {
            double v;
            long x;
            head(i, v, x);
            if (x != LONG_MAX && (list < 0 || better(v, x, best, index))) { best = v; index = x; list = i; }
        }
    };
    mine();
    for (int k = 0; k < p.n; ++k) {
        double v = best;
        long x = index;
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) {
            const double w = __shfl_xor(v, o, 64);
            const long y = __shfl_xor(x, o, 64);
            if (better(w, y, v, x)) { v = w; x = y; }
        }
        if (x == LONG_MAX) x = 0;                  // (not reached: a group has at least n candidates)
        if (x == index && list >= 0) {
            at[list] += 1;
            mine();
        }
        if (lane == 0) {
            const int r = (int)(x / p.vocab), token = (int)(x - (long)r * p.vocab);
            const long o = (long)g * p.n + k;
            p.out_scores[o] = (float)v;
            p.out_parents[o] = r;
            p.out_tokens[o] = token;
            p.out_ended[o] = token == p.eos || (p.ended != nullptr && p.ended[(long)g * p.W + r] != 0);
        }
    }
}

// ---- reordering -------------------------------------------------------------------------------------------------------------------
constexpr int REORDER_MAX = 16;
struct ReorderParams {
    char *at[REORDER_MAX];
    long stride[REORDER_MAX], bytes[REORDER_MAX];  // from a row to the next; of a row that move
    int unit[REORDER_MAX];                         // > 0: bytes of an entry, of which the first *upto move
    int strips[REORDER_MAX];                       // workgroups of the tensors before
    const int32_t *parents, *upto;
    int W, n, strip;                               // strip: bytes of a row that a workgroup has
};

// T: what a thread moves at a time (16 or 4 bytes)
template <class T>
__global__ __launch_bounds__(256) void beam_reorder_kernel(ReorderParams p) {
    extern __shared__ char raw[];
    __shared__ int32_t from[BEAM_MAX_W];
    T *lds = reinterpret_cast<T *>(raw);
    int k = 0;
    for (int i = 1; i < p.n; ++i)
        if ((int)blockIdx.x >= p.strips[i]) k = i;
    const int g = blockIdx.y, t = threadIdx.x, W = p.W;
    long bytes = p.bytes[k];
    if (p.unit[k] > 0) bytes = min(bytes, max((long)p.upto[0], 0L) * p.unit[k]);
    const long b0 = (long)((int)blockIdx.x - p.strips[k]) * p.strip;
    if (b0 >= bytes) return;
    const int per = (int)((min((long)p.strip, bytes - b0) + (long)sizeof(T) - 1) / (long)sizeof(T));      // (a row's bytes are a multiple of T)
    if (t < W) from[t] = min(max(p.parents[(long)g * W + t], 0), W - 1);
    __syncthreads();
    char *base = p.at[k] + (long)g * W * p.stride[k] + b0;
    for (int i = t; i < W * per; i += 256) {
        const int r = i / per;
        lds[i] = *reinterpret_cast<const T *>(base + r * p.stride[k] + (long)(i - r * per) * sizeof(T));
    }
    __syncthreads();
    for (int i = t; i < W * per; i += 256) {
        const int r = i / per, f = from[r];
        if (f != r) *reinterpret_cast<T *>(base + r * p.stride[k] + (long)(i - r * per) * sizeof(T)) = lds[f * per + i - r * per];
    }
}

}  // namespace smh

using namespace smh;

namespace {
struct SelectPlan { int slices, width; size_t sums, maxima, cands, bytes; };
// Slices of 8192 columns where there are rows to fill the GPU with; else of 2048, whose workgroups are done sooner
SelectPlan select_plan(long rows, int vocab, int n) {
    SelectPlan p;
    const int wide = (vocab + 8191) / 8192;
    p.width = rows * wide >= 512 ? 8192 : 2048;
    p.slices = (vocab + p.width - 1) / p.width;
    p.sums = (size_t)rows * p.slices * 8;
    p.maxima = ((size_t)rows * p.slices * 4 + 7) / 8 * 8;
    p.cands = (size_t)rows * p.slices * n * 4;
    p.bytes = p.sums + p.maxima + p.cands;
    return p;
}
bool select_sizes(int G, int W, int vocab, int n) {
    return G >= 1 && W >= 1 && W <= BEAM_MAX_W && vocab >= 1 && vocab <= (1 << 24) && n >= 1 && n <= BEAM_MAX_N && n <= vocab && (long)G * W <= (1 << 20);
}
}  // namespace

extern "C" size_t smh_beam_select_workspace_bytes(int G, int W, int vocab, int n) {
    return select_sizes(G, W, vocab, n) ? select_plan((long)G * W, vocab, n).bytes : 0;
}

extern "C" int smh_beam_select(const void *logits, long ld, const float *scores, const uint8_t *ended, int G, int W, int vocab, int n, int64_t eos, float *out_scores,
                               int32_t *out_parents, int64_t *out_tokens, uint8_t *out_ended, void *workspace, size_t workspace_bytes, smh_stream_t stream) {
    SMH_REQUIRE(W >= 1 && W <= BEAM_MAX_W, "smh_beam_select: W=%d (1 .. %d beams a group)", W, BEAM_MAX_W);
    SMH_REQUIRE(n >= 1 && n <= BEAM_MAX_N && n <= vocab, "smh_beam_select: n=%d of vocab=%d (1 .. %d, at most the vocabulary)", n, vocab, BEAM_MAX_N);
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
    const dim3 grid(plan.slices, 1, 1);
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
        if (plan.width == 8192) hipLaunchKernelGGL(beam_slice_kernel<32>, dim3(plan.slices, rows), dim3(256), 0, st, part);
        else hipLaunchKernelGGL(beam_slice_kernel<8>, dim3(plan.slices, rows), dim3(256), 0, st, part);
        if (int rc = launch_status()) return rc;
    }
    const size_t lds = (size_t)((W * plan.slices + 1) & ~1) * 4 + (size_t)W * 12;
    hipLaunchKernelGGL(beam_merge_kernel, dim3(G), dim3(64), lds, st, p);
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
    bool wide = true;
    for (int i = 0; i < n; ++i) {
        SMH_REQUIRE(tensors[i] && bytes[i] >= 0 && strides[i] >= bytes[i] && units[i] >= 0, "smh_beam_reorder: tensor %d: rows of %ld bytes %ld apart, entries of %d", i, bytes[i], strides[i],
                    units[i]);
        SMH_REQUIRE(bytes[i] % 4 == 0 && strides[i] % 4 == 0 && ((uintptr_t)tensors[i] & 3) == 0 && units[i] % 4 == 0, "smh_beam_reorder: tensor %d: rows are multiples of 4 bytes, 4-byte aligned", i);
        SMH_REQUIRE(units[i] == 0 || upto, "smh_beam_reorder: tensor %d goes by *upto, which is null", i);
        for (int j = 0; j < i; ++j) SMH_REQUIRE(tensors[i] != tensors[j], "smh_beam_reorder: tensors %d and %d are the same", j, i);
        wide = wide && bytes[i] % 16 == 0 && strides[i] % 16 == 0 && ((uintptr_t)tensors[i] & 15) == 0 && (units[i] == 0 || bytes[i] >= 0);
    }
    for (int i = 0; i < n; ++i) wide = wide && units[i] == 0;
    p.strip = wide ? 512 : 256;
    long strips = 0;
    for (int i = 0; i < n; ++i) {
        p.at[i] = (char *)tensors[i];
        p.stride[i] = strides[i];
        p.bytes[i] = bytes[i];
        p.unit[i] = units[i];
        p.strips[i] = (int)strips;
        strips += (bytes[i] + p.strip - 1) / p.strip;
        SMH_REQUIRE(strips < (1L << 31), "smh_beam_reorder: rows too long");
    }
    if (strips == 0) return 0;
    const size_t lds = (size_t)W * p.strip;
    if (wide) hipLaunchKernelGGL(beam_reorder_kernel<u32x4>, dim3((unsigned)strips, G), dim3(256), lds, (hipStream_t)stream, p);
    else hipLaunchKernelGGL(beam_reorder_kernel<uint32_t>, dim3((unsigned)strips, G), dim3(256), lds, (hipStream_t)stream, p);
    return launch_status();
}
