// The paged 8-bit cache: new rows in (with RoPE on the way), rows out.  kv8.hpp has the format.
//
// RoPE: (x1, x2) = (x[d], x[d + 64]) -> (x1 c - x2 s, x2 c + x1 s) with the fp16 table row of the token's place.  Products of two fp16 values are exact in fp32, so a
// rotated value has one rounding to fp32 and one to fp16 (which is what a row is held in), and the compiler's choice of fused operations cannot change it.
//
// All of it is bound by memory: 2 bytes in, 1 (whole blocks) or 2 (open ones) out for each value of K and V, 2 in and 2 out for each of q.
#include "kv8.hpp"

namespace smh {

struct AppendParams {
    const half_t *q, *k, *v;
    half_t *q_out;
    long q_stride, k_stride, v_stride;             // values from a token to the next; heads are contiguous
    const half_t *cos_tab, *sin_tab;
    const int32_t *lens, *cu;
    Kv8Cache c;
    int T, B, H, Hkv, max_new, table_rows;
};

// Eight dims of a row in each of 16 consecutive lanes: lane c has dims 8 c .. 8 c + 7, its partner c ^ 8 the values they are rotated with.
__device__ __forceinline__ h8 rope8(h8 x, const half_t *cos_row, const half_t *sin_row, int c) {
    const h8 cs = *reinterpret_cast<const h8 *>(cos_row + (c & 7) * 8), sn = *reinterpret_cast<const h8 *>(sin_row + (c & 7) * 8);
    const u32x4 own = __builtin_bit_cast(u32x4, x);
    u32x4 other;
#pragma unroll
    for (int i = 0; i < 4; ++i) other[i] = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)own[i], DPP_ROW_ROR8, 0xf, 0xf, false);
    const h8 y = __builtin_bit_cast(h8, other);
    const float sign = c < 8 ? -1.0f : 1.0f;
    h8 r;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        float f = (float)x[i] * (float)cs[i] + (float)y[i] * (sign * (float)sn[i]);
        asm("" : "+v"(f));                         // (two roundings wherever it stands: a mixed-precision multiply-add would have one)
        r[i] = (half_t)f;
    }
    return r;
}

__device__ __forceinline__ uint32_t abs_max8(uint32_t m, h8 x) {      // of the bit patterns: an infinity or a NaN is the largest
    const u32x4 w = __builtin_bit_cast(u32x4, x);
#pragma unroll
    for (int i = 0; i < 4; ++i) m = max(m, max(w[i] & 0x7FFFu, (w[i] >> 16) & 0x7FFFu));
    return m;
}
// The largest of 256 threads, of two numbers each.  `red`: 8 words of LDS.
__device__ __forceinline__ void block_amax(uint32_t a, uint32_t b, uint32_t *red, float &fa, float &fb) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        a = max(a, (uint32_t)__shfl_xor((int)a, o, 64));
        b = max(b, (uint32_t)__shfl_xor((int)b, o, 64));
    }
    if ((threadIdx.x & 63) == 0) {
        red[threadIdx.x >> 6] = a;
        red[4 + (threadIdx.x >> 6)] = b;
    }
    __syncthreads();
    a = max(max(red[0], red[1]), max(red[2], red[3]));
    b = max(max(red[4], red[5]), max(red[6], red[7]));
    fa = (float)__builtin_bit_cast(half_t, (uint16_t)a);
    fb = (float)__builtin_bit_cast(half_t, (uint16_t)b);
}
// (an infinity or a NaN among the values: the scale is NaN, and the block's values with it; the codes stay codes)
__device__ __forceinline__ uint32_t kv8_code(half_t x, float inverse) {
    const float r = __builtin_rintf((float)x * inverse);
    return (uint32_t)(int)(fminf(fmaxf(r, -127.0f), 127.0f) + 128.0f);
}
__device__ __forceinline__ float kv8_inverse(float amax) { return amax > 0.0f ? 127.0f / amax : 0.0f; }

constexpr int V_PITCH = 17;                        // words of LDS a line of V's codes takes: 16 and one, against bank conflicts

// Eight dims of four rows of an open V block: four places of eight lines
__device__ __forceinline__ void open_v_rows(const half_t *open_v, int quad, int dc, h8 (&x)[4]) {
    const half_t *at = open_v + dc * 8 * KV8_ROWS + kv8_place(quad * 4);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const h4 y = *reinterpret_cast<const h4 *>(at + e * KV8_ROWS);
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i][e] = y[i];
    }
}

// One block of K and V of a head becomes codes.  256 threads: thread t has rows 4 (t / 16) .. + 3 and dims 8 (t % 16) .. + 7, k[i] and v[i] of row i of them.
__device__ __forceinline__ void kv8_quantize_block(const Kv8Cache &c, long tile, const h8 (&k_rows)[4], const h8 (&v_rows)[4], uint32_t *lds, uint32_t *red) {
    const int t = threadIdx.x, quad = t >> 4, dc = t & 15;
    uint32_t mk = 0, mv = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) { mk = abs_max8(mk, k_rows[i]); mv = abs_max8(mv, v_rows[i]); }
    float ak, av;
    block_amax(mk, mv, red, ak, av);
    const float ik = kv8_inverse(ak), iv = kv8_inverse(av);
    uint8_t *k = c.k + tile * KV8_TILE;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        u32x2 w = {0, 0};
#pragma unroll
        for (int e = 0; e < 8; ++e) w[e >> 2] |= kv8_code(k_rows[i][e], ik) << (8 * (e & 3));
        *reinterpret_cast<u32x2 *>(k + (quad * 4 + i) * KV8_DIM + dc * 8) = w;
    }
    const int word = kv8_place(quad * 4) >> 2;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        uint32_t w = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) w |= kv8_code(v_rows[i][e], iv) << (8 * i);
        lds[(dc * 8 + e) * V_PITCH + word] = w;
    }
    __syncthreads();
    uint8_t *v = c.v + tile * KV8_TILE;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int at = t + i * 256, line = at >> 2, w0 = (at & 3) * 4;
        u32x4 w;
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = lds[line * V_PITCH + w0 + e];
        *reinterpret_cast<u32x4 *>(v + line * 64 + w0 * 4) = w;
    }
    if (t == 0) {
        c.scales[tile * 2] = (ak + ak * 0.0f) / 127.0f;                // (NaN for an infinity, too)
        c.scales[tile * 2 + 1] = (av + av * 0.0f) / 127.0f;
    }
}

// the page of block j of sequence b; -1: there is none
__device__ __forceinline__ long kv8_page_to_write(const Kv8Cache &c, int b, int j) {
    if (j >= c.cols) return -1;
    const long id = c.pages[(long)b * c.pages_stride + j];
    return id >= 0 && id < c.n_pages ? id : -1;
}

// One new row a sequence: a workgroup has a kv head's k, v and queries, 16 lanes each.
__global__ __launch_bounds__(256) void kv8_append_one_kernel(AppendParams p) {
    __shared__ uint32_t lds[KV8_DIM * V_PITCH];
    __shared__ uint32_t red[8];
    __shared__ h8 fresh[2][16];
    const int kvh = blockIdx.x, b = blockIdx.y;
    const Kv8Seq s = kv8_seq(p.lens, p.cu, b, p.T, 1);
    if (s.n == 0) return;
    const int t = threadIdx.x, c = t & 15, quad = t >> 4, n_rep = p.H / p.Hkv;
    auto source = [&](int r) {
        const half_t *x = r == 0 ? p.k + s.t0 * p.k_stride + kvh * KV8_DIM : r == 1 ? p.v + s.t0 * p.v_stride + kvh * KV8_DIM : p.q + s.t0 * p.q_stride + ((long)kvh * n_rep + r - 2) * KV8_DIM;
        return *reinterpret_cast<const h8 *>(x + c * 8);
    };
    h8 x = {0, 0, 0, 0, 0, 0, 0, 0};
    if (quad < n_rep + 2) x = source(quad);        // (asked for with the sequence's length, not behind it)
    const int at = min(s.old, p.table_rows - 1), row = s.old & 63;
    const half_t *cs = p.cos_tab + (long)at * 64, *sn = p.sin_tab + (long)at * 64;
    const long head = (long)b * p.Hkv + kvh;
    half_t *open_k = p.c.open_k + head * KV8_TILE, *open_v = p.c.open_v + head * KV8_TILE;
    // The 64th row of its block: the other 63 are asked for with it
    const long page = row == 63 ? kv8_page_to_write(p.c, b, s.old >> 6) : -1;
    h8 xk[4], xv[4];
    if (page >= 0) {
#pragma unroll
        for (int i = 0; i < 4; ++i) xk[i] = *reinterpret_cast<const h8 *>(open_k + (quad * 4 + i) * KV8_DIM + c * 8);
        open_v_rows(open_v, quad, c, xv);
    }
    for (int r = quad; r < n_rep + 2; r += 16) {
        if (r >= 16) x = source(r);
        if (r != 1) x = rope8(x, cs, sn, c);
        if (r >= 2) *reinterpret_cast<h8 *>(p.q_out + ((long)s.t0 * p.H + (long)kvh * n_rep + r - 2) * KV8_DIM + c * 8) = x;
        else if (row == 63) fresh[r][c] = x;
        else if ((s.old >> 6) <= p.c.cols) {
            if (r == 0) *reinterpret_cast<h8 *>(open_k + row * KV8_DIM + c * 8) = x;
            else {
                half_t *at_v = open_v + kv8_place(row);
#pragma unroll
                for (int e = 0; e < 8; ++e) at_v[(c * 8 + e) * KV8_ROWS] = x[e];
            }
        }
    }
    if (page < 0) return;
    __syncthreads();
    if (quad == 15) {
        xk[3] = fresh[0][c];
        xv[3] = fresh[1][c];
    }
    kv8_quantize_block(p.c, page * p.Hkv + kvh, xk, xv, lds, red);
}

// Any number of new rows: a workgroup has one block and kv head, or 64 new rows of one query head.
__global__ __launch_bounds__(256) void kv8_append_kernel(AppendParams p) {
    __shared__ uint32_t lds[KV8_DIM * V_PITCH];
    __shared__ uint32_t red[8];
    const int b = blockIdx.z, t = threadIdx.x, quad = t >> 4, c = t & 15;
    const Kv8Seq s = kv8_seq(p.lens, p.cu, b, p.T, p.max_new);
    if (s.n == 0) return;
    auto rotated = [&](const half_t *x, int i) {          // dims of new row i, x its first value
        const long at = min(s.old + i, p.table_rows - 1);
        return rope8(*reinterpret_cast<const h8 *>(x + c * 8), p.cos_tab + at * 64, p.sin_tab + at * 64, c);
    };
    if ((int)blockIdx.y >= p.Hkv) {
        const long h = blockIdx.y - p.Hkv;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int i = blockIdx.x * KV8_ROWS + quad * 4 + e;
            if (i < s.n) {                                // (16 lanes that rotate together agree)
                const long row = s.t0 + i;
                *reinterpret_cast<h8 *>(p.q_out + (row * p.H + h) * KV8_DIM + c * 8) = rotated(p.q + row * p.q_stride + h * KV8_DIM, i);
            }
        }
        return;
    }
    const int kvh = blockIdx.y, total = kv8_kept(s.old + s.n, p.c.cols), first = s.old >> 6, j = first + blockIdx.x, open = total >> 6;
    if (j > open) return;
    const long head = (long)b * p.Hkv + kvh;
    half_t *open_k = p.c.open_k + head * KV8_TILE, *open_v = p.c.open_v + head * KV8_TILE;
    const half_t *k = p.k + (long)s.t0 * p.k_stride + kvh * KV8_DIM, *v = p.v + (long)s.t0 * p.v_stride + kvh * KV8_DIM;
    // the new rows among the total % 64 of the block that stays open
    auto leave_open = [&]() {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int row = quad * 4 + e, i = open * KV8_ROWS + row - s.old;
            if (row >= (total & 63) || i < 0) continue;
            *reinterpret_cast<h8 *>(open_k + row * KV8_DIM + c * 8) = rotated(k + i * p.k_stride, i);
            const h8 x = *reinterpret_cast<const h8 *>(v + i * p.v_stride + c * 8);
            const int place = kv8_place(row);
#pragma unroll
            for (int d = 0; d < 8; ++d) open_v[(c * 8 + d) * KV8_ROWS + place] = x[d];
        }
    };
    // The first block may need open rows of before, whose places the last one's take: then one workgroup has both, in this order
    const bool both = (s.old & 63) != 0 && open > first;
    if (j == open) {
        if (!both) leave_open();
        return;
    }
    const long page = kv8_page_to_write(p.c, b, j);
    if (page >= 0) {
        const int before = s.old - j * KV8_ROWS;          // rows of the block that were there
        h8 xk[4], xv[4];
        if (quad * 4 < before) open_v_rows(open_v, quad, c, xv);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int r = quad * 4 + e;
            const long i = r - before;
            if (i < 0) xk[e] = *reinterpret_cast<const h8 *>(open_k + r * KV8_DIM + c * 8);
            else {
                xk[e] = rotated(k + i * p.k_stride, (int)i);
                xv[e] = *reinterpret_cast<const h8 *>(v + i * p.v_stride + c * 8);
            }
        }
        kv8_quantize_block(p.c, page * p.Hkv + kvh, xk, xv, lds, red);
    }
    if (both && blockIdx.x == 0) {
        __syncthreads();
        leave_open();
    }
}

struct RowsParams {
    half_t *k, *v;                                 // [B][count][Hkv][128]
    const int32_t *total, *first;
    Kv8Cache c;
    int B, Hkv, count;
};

// Rows as the cache holds them, in fp16: a workgroup has a block and kv head.  Reads 1 (or 2), writes 2 bytes a value.
__global__ __launch_bounds__(256) void kv8_rows_kernel(RowsParams p) {
    const int kvh = blockIdx.y, b = blockIdx.z, t = threadIdx.x, quad = t >> 4, dc = t & 15;
    const int first = min(max(p.first[b], 0), KV8_MAX_LEN), total = kv8_kept(min(max(p.total[b], 0), KV8_MAX_LEN), p.c.cols);
    const int j = (first >> 6) + blockIdx.x, whole = total >> 6;
    const int row0 = j * KV8_ROWS + quad * 4;
    if (j * KV8_ROWS >= first + p.count) return;
    const long head = (long)b * p.Hkv + kvh;
    h8 k[4], v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) k[i] = v[i] = h8{0, 0, 0, 0, 0, 0, 0, 0};
    const int place = kv8_place(quad * 4);
    if (j < whole) {
        const long page = min(max((long)p.c.pages[(long)b * p.c.pages_stride + j], 0L), p.c.n_pages - 1), tile = page * p.Hkv + kvh;
        const float ks = p.c.scales[tile * 2], vs = p.c.scales[tile * 2 + 1];
        const uint8_t *kt = p.c.k + tile * KV8_TILE, *vt = p.c.v + tile * KV8_TILE;
        u32x2 kw[4];
        uint32_t vw[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) kw[i] = *reinterpret_cast<const u32x2 *>(kt + (quad * 4 + i) * KV8_DIM + dc * 8);
#pragma unroll
        for (int e = 0; e < 8; ++e) vw[e] = *reinterpret_cast<const uint32_t *>(vt + (dc * 8 + e) * KV8_ROWS + place);
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                float a = (float)((int)((kw[i][e >> 2] >> (8 * (e & 3))) & 255) - 128) * ks, c = (float)((int)((vw[e] >> (8 * i)) & 255) - 128) * vs;
                asm("" : "+v"(a), "+v"(c));        // (to fp32 first, as everywhere)
                k[i][e] = (half_t)a;
                v[i][e] = (half_t)c;
            }
    } else if (j == whole) {
        const half_t *kt = p.c.open_k + head * KV8_TILE, *vt = p.c.open_v + head * KV8_TILE;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (row0 + i < total) k[i] = *reinterpret_cast<const h8 *>(kt + (quad * 4 + i) * KV8_DIM + dc * 8);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const h4 x = *reinterpret_cast<const h4 *>(vt + (dc * 8 + e) * KV8_ROWS + place);
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (row0 + i < total) v[i][e] = x[i];
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int at = row0 + i - first;
        if (at < 0 || at >= p.count) continue;
        const long o = (((long)b * p.count + at) * p.Hkv + kvh) * KV8_DIM + dc * 8;
        *reinterpret_cast<h8 *>(p.k + o) = k[i];
        *reinterpret_cast<h8 *>(p.v + o) = v[i];
    }
}

}  // namespace smh

using namespace smh;

namespace {
bool aligned16(const void *p) { return ((uintptr_t)p & 15) == 0; }
// what all entry points ask of a cache; 0, or -1 with the error set
int cache_ok(const char *who, const void *k, const void *v, const void *scales, const void *open_k, const void *open_v, const int32_t *pages, long n_pages, long stride, int cols,
             int B, int Hkv, int D) {
    SMH_REQUIRE(D == KV8_DIM, "%s: head dim %d (only 128)", who, D);
    SMH_REQUIRE(B >= 1 && B <= 65535 && Hkv >= 1 && Hkv <= 4096, "%s: B=%d (1 .. 65535) Hkv=%d (1 .. 4096)", who, B, Hkv);
    SMH_REQUIRE(k && v && scales && open_k && open_v && pages, "%s: null pointer in the cache", who);
    SMH_REQUIRE(aligned16(k) && aligned16(v) && aligned16(open_k) && aligned16(open_v) && ((uintptr_t)scales & 7) == 0, "%s: the cache's tensors are 16-byte aligned, its scales 8", who);
    SMH_REQUIRE(n_pages >= 1 && cols >= 0 && cols <= KV8_MAX_LEN / KV8_ROWS - 1 && stride >= cols, "%s: n_pages=%ld pages_cols=%d (at most %d) pages_stride=%ld", who, n_pages, cols,
                KV8_MAX_LEN / KV8_ROWS - 1, stride);
    return 0;
}
}  // namespace

extern "C" int smh_kv8_append(const void *q, const void *k, const void *v, void *q_out, int T, int B, int H, int Hkv, int D, long q_stride, long k_stride, long v_stride,
                              const void *cos_tab, const void *sin_tab, int table_rows, const int32_t *lens, const int32_t *cu, int max_new, void *codes_k, void *codes_v, void *scales,
                              void *open_k, void *open_v, const int32_t *pages, long n_pages, long pages_stride, int pages_cols, smh_stream_t stream) {
    if (cache_ok("smh_kv8_append", codes_k, codes_v, scales, open_k, open_v, pages, n_pages, pages_stride, pages_cols, B, Hkv, D)) return -1;
    SMH_REQUIRE(H >= 1 && H % Hkv == 0 && H + Hkv <= 65535, "smh_kv8_append: H=%d Hkv=%d", H, Hkv);
    SMH_REQUIRE(T >= 0 && max_new >= 0 && max_new <= KV8_MAX_LEN && table_rows >= 1, "smh_kv8_append: T=%d max_new=%d table_rows=%d", T, max_new, table_rows);
    SMH_REQUIRE(cu || (T == B && max_new == 1), "smh_kv8_append: without cu every sequence has one row: T=%d B=%d max_new=%d", T, B, max_new);
    SMH_REQUIRE(q_stride >= (long)H * D && k_stride >= (long)Hkv * D && v_stride >= (long)Hkv * D && q_stride % 8 == 0 && k_stride % 8 == 0 && v_stride % 8 == 0,
                "smh_kv8_append: token strides %ld %ld %ld", q_stride, k_stride, v_stride);
    if (T == 0 || max_new == 0) return 0;
    SMH_REQUIRE(q && k && v && q_out && cos_tab && sin_tab && lens, "smh_kv8_append: null pointer");
    SMH_REQUIRE(aligned16(q) && aligned16(k) && aligned16(v) && aligned16(q_out) && aligned16(cos_tab) && aligned16(sin_tab), "smh_kv8_append: tensors are 16-byte aligned");
    AppendParams p{(const half_t *)q, (const half_t *)k, (const half_t *)v, (half_t *)q_out, q_stride, k_stride, v_stride, (const half_t *)cos_tab, (const half_t *)sin_tab, lens, cu,
                   {(uint8_t *)codes_k, (uint8_t *)codes_v, (float *)scales, (half_t *)open_k, (half_t *)open_v, pages, pages_stride, n_pages, pages_cols},
                   T, B, H, Hkv, cu ? max_new : 1, table_rows};
    if (p.max_new == 1) hipLaunchKernelGGL(kv8_append_one_kernel, dim3(Hkv, B), dim3(256), 0, (hipStream_t)stream, p);
    else {
        const int most = min(p.max_new, T);
        hipLaunchKernelGGL(kv8_append_kernel, dim3((most + 62) / KV8_ROWS + 1, Hkv + H, B), dim3(256), 0, (hipStream_t)stream, p);
    }
    return launch_status();
}

extern "C" int smh_kv8_rows(void *out_k, void *out_v, int B, int Hkv, int D, const int32_t *total, const int32_t *first, int count, const void *codes_k, const void *codes_v,
                            const void *scales, const void *open_k, const void *open_v, const int32_t *pages, long n_pages, long pages_stride, int pages_cols, smh_stream_t stream) {
    if (cache_ok("smh_kv8_rows", codes_k, codes_v, scales, open_k, open_v, pages, n_pages, pages_stride, pages_cols, B, Hkv, D)) return -1;
    SMH_REQUIRE(count >= 0 && count <= KV8_MAX_LEN, "smh_kv8_rows: count=%d", count);
    if (count == 0) return 0;
    SMH_REQUIRE(out_k && out_v && total && first, "smh_kv8_rows: null pointer");
    SMH_REQUIRE(aligned16(out_k) && aligned16(out_v), "smh_kv8_rows: tensors are 16-byte aligned");
    RowsParams p{(half_t *)out_k, (half_t *)out_v, total, first,
                 {(uint8_t *)codes_k, (uint8_t *)codes_v, (float *)scales, (half_t *)open_k, (half_t *)open_v, pages, pages_stride, n_pages, pages_cols}, B, Hkv, count};
    hipLaunchKernelGGL(kv8_rows_kernel, dim3((count + 62) / KV8_ROWS + 1, Hkv, B), dim3(256), 0, (hipStream_t)stream, p);
    return launch_status();
}
