// The paged 8-bit cache: what its kernels share.
//
// A block is 64 consecutive rows of a sequence.  For each kv head a whole block holds codes u = rint(x * 127 / amax) + 128 (one byte, 1 .. 255) and the
// scale amax / 127 (fp32) of K and of V; x is worth (u - 128) * scale.  The block that is not whole yet - the open one, one for each sequence - is held
// in fp16 and becomes codes when its 64th row arrives: every row is quantised once, with the largest value of its block known, and what a cache
// holds does not depend on the calls that its rows came in.
//
// Both orders are those in which the lanes of the attention take their MFMA operands (v_mfma_f32_16x16x32_f16: lane l has row or column l % 16 and the k
// values 8 (l / 16) ..): K is [row][dim]; V is [dim][place], place 16 g + 8 u + 4 j + i being row 32 u + 16 j + 4 g + i of the block (i, g < 4, u, j < 2).  The
// scores of a 16-row tile leave the first product with rows 4 g .. 4 g + 3 in lane group g, so two tiles are the eight probabilities that lane group g gives the
// second product, and they meet eight consecutive places of V: nothing crosses lanes between the two.
#pragma once

#include "smh_common.hpp"

namespace smh {

constexpr int KV8_ROWS = 64;                       // rows of a block
constexpr int KV8_DIM = 128;
constexpr int KV8_TILE = KV8_ROWS * KV8_DIM;       // bytes of K or V of a block and head, values of an open one
constexpr int KV8_MAX_LEN = 1 << 29;

struct Kv8Cache {
    uint8_t *k, *v;                                // [n_pages][Hkv][64][128], [n_pages][Hkv][128][64]
    float *scales;                                 // [n_pages][Hkv][2]
    half_t *open_k, *open_v;                       // [B][Hkv][64][128], [B][Hkv][128][64]
    const int32_t *pages;                          // [B][pages_stride], `cols` of them in use
    long pages_stride, n_pages;
    int cols;
};

// A sequence's part in a call: its new rows are rows t0 .. t0 + n - 1 of the packed tensors and places old .. old + n - 1 of the sequence.  What the
// caller's numbers say beyond the tensors is cut: nothing is read or written outside them.
struct Kv8Seq { int t0, n, old; };
__device__ __forceinline__ Kv8Seq kv8_seq(const int32_t *lens, const int32_t *cu, int b, int T, int max_new) {
    int t0 = b, t1 = b + 1;
    if (cu != nullptr) {
        t0 = min(max(cu[b], 0), T);
        t1 = min(max(cu[b + 1], t0), T);
    }
    return Kv8Seq{t0, min(t1 - t0, max_new), min(max(lens[b], 0), KV8_MAX_LEN)};
}

// Rows that a cache keeps of a sequence of `length`: the table's blocks and 63 of the open one behind them.  A length that is 64 and more past these is taken for a wrong one: it
// has the table's blocks alone.
__device__ __forceinline__ int kv8_kept(int length, int cols) {
    return length < (cols + 2) * KV8_ROWS ? min(length, cols * KV8_ROWS + KV8_ROWS - 1) : cols * KV8_ROWS;
}

// place of row r of a block in a line of V
__device__ __forceinline__ int kv8_place(int r) { return ((r >> 2) & 3) * 16 + (r >> 5) * 8 + ((r >> 4) & 1) * 4 + (r & 3); }

// Four codes as fp16 integers -127 .. 127: the byte u in the low bits of fp16 1024 is 1024 + u, and 1152 less is exact.
__device__ __forceinline__ void kv8_codes4(uint32_t w, h2 &a, h2 &b) {
    const h2 off = {(half_t)-1152.0f, (half_t)-1152.0f};
    a = as_h2(__builtin_amdgcn_perm(0x64646464u, w, 0x04010400u)) + off;
    b = as_h2(__builtin_amdgcn_perm(0x64646464u, w, 0x04030402u)) + off;
}
__device__ __forceinline__ h8 kv8_codes8(uint32_t w0, uint32_t w1) {
    h2 a, b, c, d;
    kv8_codes4(w0, a, b);
    kv8_codes4(w1, c, d);
    return h8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

}  // namespace smh
