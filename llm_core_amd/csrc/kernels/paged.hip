// paged.hip — a cache of K/V pages that several continuations of a text share:
// attention over it, the store of new rows, the fork of page tables, the
// compaction after a drafted tree was verified (include/axf_hip.h has the layout
// and the calls' rules).
#include "common.hpp"
#include "paged_index.hpp"

#include <type_traits>

namespace axf {

namespace {

constexpr float kLog2e = 1.44269504088896340736f;

// The token counts of sequence s, cut to what the call and the table can hold.
struct SeqLen {
    int held, tok;
};
__device__ __forceinline__ SeqLen seq_len(const int* len, const int* n_tok, int max_tok, int s,
                                          int table_ld, int page_shift) {
    SeqLen n;
    n.held = kv_len(len[s], table_ld, page_shift);
    n.tok = n_tok ? min(max(n_tok[s], 0), max_tok) : max_tok;
    return n;
}

// q element d of row `row`, head h: bias, RoPE (rotate-half), times 1/sqrt(HD).
template <int HD>
__device__ __forceinline__ float q_value(const PagedArgs& a, long row, int h, int d) {
    const float* qr = a.q + row * a.q_ld + h * HD;
    float x = qr[d];
    if (a.bq) x += a.bq[h * HD + d];
    if (a.pos) {
        const int half = HD / 2, e = d < half ? d + half : d - half, f = d < half ? d : e;
        float y = qr[e];
        if (a.bq) y += a.bq[h * HD + e];
        const long p = min(max(a.pos[row], 0), a.n_pos - 1);
        const float c = a.cos_t[p * half + f], w = a.sin_t[p * half + f];
        x = d < half ? x * c - y * w : x * c + y * w;
    }
    return x;
}

// ---- attention ------------------------------------------------------------------
// A sequence's tokens and the query heads of one KV head are rows of one matrix:
// row rho = i * G + h of token i, head kvh * G + h.  S^T = K Q^T and O^T = V^T P^T on
// the matrix cores (16x16x32), the softmax online: a running maximum m and sum l a
// row, in base 2 (t = s * log2(e) / sqrt(HD)).  With the products transposed a lane
// keeps one query row (its column, lane & 15) through both: S^T leaves it 4 keys of a
// 16-key tile (4 (lane >> 4) + r), two tiles are the 8 keys that the second product's
// B operand wants of a lane, so P never leaves its lane, and rescaling O needs no
// exchange either.
//
// fp32 is kept on 16-bit operands by splitting:
//   F32 pages: x = h + m + l, three bf16 cut off one after the other (8 bits each: exact
//   down to 2^-110, below it to bf16's smallest step, 2^-133), and six of the nine products:
//   hh, hm, mh, mm, hl, lh (the other three are below 2^-21 of |x y|, 2^-24 as a rule);
//   6/16 of the fp32 matrix rate's time.
//   F16 pages: K and V are fp16 as they are; q (scaled by a power of two a row) is
//   h + 2^-12 l, two fp16 parts with a sum of their own each, 22 bits of every element;
//   p (times 2^15) is h + l with one sum, 22 bits down to p = 2^-16 and 2^-39 below
//   (a second sum would cost O's registers again): two products, no work on K or V.
//   A subnormal value (below 2^-14) counts with the exponent -14 where products are
//   aligned, so what is below 2^-37 of O (2^-23 of that exponent) is cut off there.
// Infinities and NaN do not split, and 0 times one of them in a masked place is NaN: a
// row whose result is not finite is done again in plain fp32 (row_careful, by the
// joining kernel), where masked places are left out.  So is a row whose scores are too
// far out (far_out) or, with F32 pages, whose q has elements that 2^-133 is not small
// beside (q_splits): their results are made NaN.  And, with F32 pages, one with an element
// below kSmall, where V's lost digits would show.

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4_a4 __attribute__((ext_vector_type(4), aligned(4)));

constexpr int kStep = 32;  // keys a step: two 16-key tiles

__device__ __forceinline__ uint32_t pack_hi(float lo, float hi) {
    return __builtin_amdgcn_perm(__float_as_uint(hi), __float_as_uint(lo), 0x07060302u);
}
__device__ __forceinline__ float cut_bf16(float x) {
    return __uint_as_float(__float_as_uint(x) & 0xffff0000u);
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
    const _Float16 a = (_Float16)lo, b = (_Float16)hi;
    uint16_t x, y;
    __builtin_memcpy(&x, &a, 2);
    __builtin_memcpy(&y, &b, 2);
    return (uint32_t)x | ((uint32_t)y << 16);
}

// How values of a page type become 16-bit operands.  KP / QP: parts of K and V, of q
// and p; SUMS: accumulators of q's product; kUp: what O is too large by.
template <class T>
struct Parts;

template <>
struct Parts<float> {
    static constexpr int KP = 3, QP = 3, SUMS = 1;
    static constexpr float kUp = 1.f;
    static constexpr bool kScaleQ = false;
    static __device__ __forceinline__ void split(const float (&x)[8], uint4 (&f)[3]) {
        uint32_t w[3][4];
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const float a = x[2 * e], b = x[2 * e + 1];
            const float a1 = a - cut_bf16(a), b1 = b - cut_bf16(b);
            const float a2 = a1 - cut_bf16(a1), b2 = b1 - cut_bf16(b1);
            w[0][e] = pack_hi(a, b);
            w[1][e] = pack_hi(a1, b1);
            w[2][e] = pack_hi(a2, b2);
        }
#pragma unroll
        for (int p = 0; p < 3; p++) f[p] = make_uint4(w[p][0], w[p][1], w[p][2], w[p][3]);
    }
    static __device__ __forceinline__ void split_q(const float (&x)[8], uint4 (&f)[3]) { split(x, f); }
    static __device__ __forceinline__ void split_p(const float (&x)[8], uint4 (&f)[3]) { split(x, f); }
    static __device__ __forceinline__ void split_kv(const float (&x)[8], uint4 (&f)[3]) { split(x, f); }
    static __device__ __forceinline__ f32x4 mul(const uint4& a, const uint4& b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a),
                                                       __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    }
    // c[i][j] += a[i] b[j], NA x NB products side by side (the six sums of one wait for
    // each other), the smallest first
    template <int NA, int NB>
    static __device__ __forceinline__ void product(const uint4 (&a)[NA][3], const uint4* const (&b)[NB],
                                                   f32x4* const (&c)[NA][NB]) {
        constexpr int A[6] = {2, 0, 1, 1, 0, 0}, B[6] = {0, 2, 1, 0, 1, 0};
#pragma unroll
        for (int p = 0; p < 6; p++)
#pragma unroll
            for (int i = 0; i < NA; i++)
#pragma unroll
                for (int j = 0; j < NB; j++) *c[i][j] = mul(a[i][A[p]], b[j][B[p]], *c[i][j]);
    }
    // the same for scores, whose sums are SUMS apart
    template <int NA, int NB>
    static __device__ __forceinline__ void scores(const uint4 (&a)[NA][3], const uint4* const (&b)[NB],
                                                  f32x4* const (&c)[NA][NB]) {
        product<NA, NB>(a, b, c);
    }
    static __device__ __forceinline__ float total(const f32x4 (&c)[1], int r) { return c[0][r]; }
};

template <>
struct Parts<_Float16> {
    static constexpr int KP = 1, QP = 2, SUMS = 2;
    static constexpr float kUp = 32768.f;
    static constexpr bool kScaleQ = true;
    static __device__ __forceinline__ void split(const float (&x)[8], float low, uint4 (&f)[2]) {
        uint32_t h[4], l[4];
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const float a = x[2 * e], b = x[2 * e + 1];
            const float a0 = (float)(_Float16)a, b0 = (float)(_Float16)b;
            h[e] = pack_f16(a, b);
            l[e] = pack_f16((a - a0) * low, (b - b0) * low);
        }
        f[0] = make_uint4(h[0], h[1], h[2], h[3]);
        f[1] = make_uint4(l[0], l[1], l[2], l[3]);
    }
    static __device__ __forceinline__ void split_q(const float (&x)[8], uint4 (&f)[2]) {
        split(x, 4096.f, f);
    }
    static __device__ __forceinline__ void split_p(const float (&x)[8], uint4 (&f)[2]) {
        float y[8];
#pragma unroll
        for (int e = 0; e < 8; e++) y[e] = x[e] * kUp;
        split(y, 1.f, f);
    }
    static __device__ __forceinline__ f32x4 mul(const uint4& a, const uint4& b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a),
                                                      __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    }
    template <int NA, int NB>
    static __device__ __forceinline__ void product(const uint4 (&a)[NA][1], const uint4* const (&b)[NB],
                                                   f32x4* const (&c)[NA][NB]) {
#pragma unroll
        for (int p = 1; p >= 0; p--)
#pragma unroll
            for (int i = 0; i < NA; i++)
#pragma unroll
                for (int j = 0; j < NB; j++) *c[i][j] = mul(a[i][0], b[j][p], *c[i][j]);
    }
    template <int NA, int NB>
    static __device__ __forceinline__ void scores(const uint4 (&a)[NA][1], const uint4* const (&b)[NB],
                                                  f32x4* const (&c)[NA][NB]) {
#pragma unroll
        for (int p = 0; p < 2; p++)
#pragma unroll
            for (int i = 0; i < NA; i++)
#pragma unroll
                for (int j = 0; j < NB; j++) c[i][j][p] = mul(a[i][0], b[j][p], c[i][j][p]);
    }
    static __device__ __forceinline__ float total(const f32x4 (&c)[2], int r) {
        return fmaf(c[1][r], 1.f / 4096.f, c[0][r]);
    }
};

// A weight is exp2(s c - m), its product not rounded but m, the largest one, rounded to
// fp32: all of a row's weights are too large or small by one factor, 2^(half a step of m)
// at the most, which their sum takes out again.  Up to |m| = 2^22 it is 2^0.25; from 2^28
// on it leaves fp16 parts without digits, from 2^31 on weights without any.  top: the row's
// largest score (base 2), -inf where it sees nothing.
__device__ __forceinline__ bool far_out(float top) {
    return fabsf(top) > 4194304.f && top != -INFINITY;
}

// Whether F32 pages' three parts hold a score's digits: q's elements are 0 or from 2^-100 to
// 2^100, so that its own last steps, and 2^-133 of a key's element times it, are below
// 2^-33.  high: the largest |element|; low: the least of their bits less one (of 0: all ones).
__device__ __forceinline__ bool q_splits(float high, uint32_t low) {
    return high <= 0x1p100f && low >= 0x0d7fffffu;  // 2^-100 is 0x0d800000
}
constexpr float kSmall = 0x1p-100f;

// Reductions over the four 16-lane rows of a wave (lanes n, n + 16, n + 32, n + 48),
// every lane receiving the result.  v_permlane{16,32}_swap of a value with itself
// leaves it beside its partner rows' value.
__device__ __forceinline__ float rows_max(float x) {
    auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float rows_sum(float x) {
    auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

__device__ __forceinline__ void load8(const float* p, float (&v)[8]) {
    const f32x4_a4 u = *reinterpret_cast<const f32x4_a4*>(p);
    const f32x4_a4 w = *reinterpret_cast<const f32x4_a4*>(p + 4);
#pragma unroll
    for (int e = 0; e < 4; e++) {
        v[e] = u[e];
        v[4 + e] = w[e];
    }
}

// q elements d .. d+7 and HD/2 + d .. (d % 8 == 0, d < HD/2) of a row, which RoPE turns
// into each other: bias and RoPE by the tables' row pos.
template <int HD>
__device__ __forceinline__ void q_values8(const PagedArgs& a, long row, int h, int d, long pos,
                                          float (&x)[8], float (&y)[8]) {
    constexpr int half = HD / 2;
    const float* qr = a.q + row * a.q_ld + h * HD + d;
    load8(qr, x);
    load8(qr + half, y);
    if (a.bq) {
        float b[8], b2[8];
        load8(a.bq + h * HD + d, b);
        load8(a.bq + h * HD + d + half, b2);
#pragma unroll
        for (int e = 0; e < 8; e++) {
            x[e] += b[e];
            y[e] += b2[e];
        }
    }
    if (a.pos) {
        float c[8], s[8];
        load8(a.cos_t + pos * half + d, c);
        load8(a.sin_t + pos * half + d, s);
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const float u = x[e], w = y[e];
            x[e] = fmaf(u, c[e], -(w * s[e]));
            y[e] = fmaf(w, c[e], u * s[e]);
        }
    }
}
// The row's position in the RoPE tables.
__device__ __forceinline__ long q_pos(const PagedArgs& a, long row) {
    return a.pos ? min(max(a.pos[row], 0), a.n_pos - 1) : 0;
}

// How the work is split.  A part is one sequence's, KV head's and row tile's walk over
// its keys, in units of `per` steps; all parts' units in a row are dealt out evenly to
// the grid's workgroups, which are as many as run at once: every workgroup has the same
// number of units, however ragged the lengths, and a part that lies in one share is
// finished there.  A share holds at most two unfinished ends (its first part's and its
// last's); they go to the workgroup's two slots of partial sums, which
// k_attn_paged_join adds.
constexpr int kPlanSeqs = 256;  // sequences a launch

// a / b of whole numbers, a >= 0, b > 0, a / b < 2^50: hardware has no 64-bit integer
// division, and a correctly rounded one in doubles is 35 instructions.  1 / b from the
// approximation (2^-23 or better) in two Newton steps is good to 2^-51, so the product's
// whole part is off by one at the most.
__device__ __forceinline__ long div_whole(long a, long b) {
    const double d = (double)b;
    double y = __builtin_amdgcn_rcp(d);
    y = fma(fma(-d, y, 1.), y, y);
    y = fma(fma(-d, y, 1.), y, y);
    const long q = (long)((double)a * y);
    const long r = a - q * b;
    return r < 0 ? q - 1 : (r >= b ? q + 1 : q);
}

// A unit is `per` steps of 32 keys.  With per 3 a last tile at most half full has units of
// 4 steps: its waves without rows leave the others the SIMDs, and a step takes 0.74 of a
// full tile's time (16 sequences @8000, 64 and 128 rows: 275 and 368 us).  48 tokens of 16
// sequences @8000 (192 rows), with 4 and with 3 steps: 128 elements a head F32 592 and 610 us,
// F16 327 and 356; 64 elements F32 375 and 412; 256 elements F16 259 and 266, F32 904 and
// 892 (@2000: 253 and 260).
struct SeqWork {
    int rows, tiles, per_last;
    long units, last;  // of a part, of one of the last row tile
    __device__ __forceinline__ long of_head() const { return (tiles - 1) * units + last; }
};
__device__ __forceinline__ long units_of(uint32_t steps, int per) {
    return per == 3 ? (steps + 2) / 3 : (steps + per - 1) >> __builtin_ctz(per);
}
// tile_rows is a power of two
__device__ __forceinline__ SeqWork seq_work(const SeqLen& n, int G, int tile_rows, int per) {
    SeqWork w;
    w.rows = n.tok * G;
    w.tiles = (w.rows + tile_rows - 1) >> __builtin_ctz(tile_rows);
    const int over = w.rows & (tile_rows - 1);
    w.per_last = per == 3 && over && over <= tile_rows / 2 ? 4 : per;
    const uint32_t steps = ((uint32_t)n.held + n.tok + kStep - 1) / kStep;
    w.units = w.tiles ? units_of(steps, per) : 0;
    w.last = w.tiles ? units_of(steps, w.per_last) : 0;
    return w;
}

// cum[s]: units before sequence s (cum[n_seq]: all), and its lengths; the first 256
// threads.
__device__ __forceinline__ void make_plan(const PagedArgs& a, int tile_rows, long* cum,
                                          long* part, SeqLen* lens) {
    const int t = threadIdx.x, lane = t & 63;
    long w = 0;
    if (t < a.n_seq) {
        const SeqLen n = seq_len(a.len, a.n_tok, a.max_tok, t, a.table_ld, a.page_shift);
        lens[t] = n;
        const SeqWork k = seq_work(n, a.group, tile_rows, a.per);
        w = k.of_head() * a.n_kv_heads;
    }
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const long y = __shfl_up(w, off, 64);
        if (lane >= off) w += y;
    }
    if (lane == 63 && t < kPlanSeqs) part[t >> 6] = w;
    __syncthreads();
    if (t < kPlanSeqs) {
        for (int i = 0; i < (t >> 6); i++) w += part[i];
        cum[t + 1] = w;
    }
    if (t == 0) cum[0] = 0;
    __syncthreads();
}

// Shares that have units (none is empty before the last), the first unit of share w of
// n, and the share that unit u is in.
__device__ __forceinline__ int shares_used(const PagedArgs& a, long total) {
    return (int)min((long)a.shares, total);
}
__device__ __forceinline__ long share_start(long total, int w, int n) {
    return div_whole(total * w, n);
}
__device__ __forceinline__ int share_of(long total, long u, int n) {
    return (int)div_whole((u + 1) * n - 1, total);
}

__device__ __forceinline__ long uniform(long x) {
    return (long)(((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(x >> 32)) << 32) |
                  (uint32_t)__builtin_amdgcn_readfirstlane((int)x));
}

// One part's stretch of keys in a share.
struct Span {
    int s, held, tok, j0, j1;
    const int* table;
    int rows, kvh, tile;
    int slot;  // of partial sums, -1: the whole part
};

// The stretch at unit lo of a share that ends at hi; moves lo behind it.
__device__ __forceinline__ Span next_span(const PagedArgs& a, const long* cum, const SeqLen* lens,
                                          int tile_rows, int share, int& s, long& lo, long hi) {
    // sequences whose units end at lo or before, 64 at a time
    for (;;) {
        const int t = s + (threadIdx.x & 63);
        const int n = __popcll(__ballot(t < a.n_seq && cum[t + 1] <= lo));
        s += n;
        if (n < 64) break;
    }
    Span p;
    p.s = s;
    SeqLen n = lens[s];
    n.held = __builtin_amdgcn_readfirstlane(n.held);
    n.tok = __builtin_amdgcn_readfirstlane(n.tok);
    const SeqWork w = seq_work(n, a.group, tile_rows, a.per);
    p.held = n.held;
    p.tok = n.tok;
    p.rows = w.rows;
    p.table = a.table + (long)p.s * a.table_ld;
    const long at = lo - uniform(cum[p.s]), head = uniform(div_whole(at, w.of_head()));
    const long in = at - head * w.of_head();
    p.kvh = (int)head;
    p.tile = w.tiles > 1 ? min((int)uniform(div_whole(in, w.units)), w.tiles - 1) : 0;
    const bool end = p.tile == w.tiles - 1;
    const long n_units = end ? w.last : w.units;
    const int keys = (end ? w.per_last : a.per) * kStep;  // of a unit
    const long u0 = in - p.tile * w.units, u1 = min(n_units, u0 + hi - lo);
    p.j0 = __builtin_amdgcn_readfirstlane((int)(u0 * keys));
    p.j1 = __builtin_amdgcn_readfirstlane((int)min(u1 * keys, (long)n.held + n.tok));
    p.slot = u0 > 0 ? 2 * share : (u1 < n_units ? 2 * share + 1 : -1);
    lo += u1 - u0;
    return p;
}

__device__ __forceinline__ uint64_t seen_mask(const PagedArgs& a, long row, int i) {
    return a.mask ? a.mask[row] : ~0ull >> (63 - i);
}

// One query row in plain fp32, a wave over the head's elements (o: elements
// E lane ..), four keys at a time.
template <int HD, class T>
__device__ __forceinline__ void row_careful(const PagedArgs& a, int s, int i, int h, float (&y)[HD / 64]) {
    constexpr int E = HD / 64, U = 4;
    const int lane = threadIdx.x & 63, kvh = h / a.group;
    const long row = (long)s * a.max_tok + i, ld = (long)a.n_kv_heads * HD;
    const SeqLen n = seq_len(a.len, a.n_tok, a.max_tok, s, a.table_ld, a.page_shift);
    const int* table = a.table + (long)s * a.table_ld;
    const uint64_t mask = seen_mask(a, row, i);
    const T* k = static_cast<const T*>(a.k) + kvh * HD + lane * E;
    const T* v = static_cast<const T*>(a.v) + kvh * HD + lane * E;
    const float c = kLog2e / sqrtf((float)HD);
    float q[E], o[E];
#pragma unroll
    for (int e = 0; e < E; e++) {
        q[e] = q_value<HD>(a, row, h, lane * E + e);
        o[e] = 0.f;
    }
    float m = -INFINITY, l = 0.f;
    const int total = n.held + n.tok;
    for (int j0 = 0; j0 < total; j0 += U) {
        float d[U], w[U][E];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int j = min(j0 + u, total - 1);
            const long r = kv_row(j, table, a.table_ld, a.n_pages, a.page_shift);
            const bool see = j0 + u < total && r >= 0 &&
                             (j < n.held || ((mask >> (j - n.held)) & 1));
            float x = 0.f;
#pragma unroll
            for (int e = 0; e < E; e++) {
                x = fmaf(q[e], (float)k[max(r, 0L) * ld + e], x);
                w[u][e] = (float)v[max(r, 0L) * ld + e];
            }
            x = wave_sum(x) * c;
            d[u] = see ? x : -INFINITY;
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            if (d[u] == -INFINITY) continue;  // no weight, whatever the value
            const float mn = fmaxf(m, d[u]);
            const float base = mn == -INFINITY ? 0.f : mn;
            const float keep = exp2f(m - base), p = exp2f(d[u] - base);
            l = l * keep + p;
#pragma unroll
            for (int e = 0; e < E; e++) o[e] = fmaf(p, w[u][e], keep == 0.f ? 0.f : o[e] * keep);
            m = mn;
        }
    }
#pragma unroll
    for (int e = 0; e < E; e++) y[e] = l == 0.f ? 0.f : o[e] / l;
}

// q's fragments of one 16-row tile: lane's row, elements 32 c + 8 (lane >> 4) .. +7 of
// each 32-element chunk.  A row past the last takes the first's values (its results go
// nowhere).  scale: what scores are multiplied by (with F16 pages the row was scaled to
// the top of fp16's range).
template <int HD, class T>
__device__ __forceinline__ void load_q(const PagedArgs& a, const Span& sp, int rho, long pos,
                                       uint4 (&qf)[HD / 32][Parts<T>::QP], float& scale) {
    constexpr int NC = HD / 32;
    const int g = (threadIdx.x & 63) >> 4, i = rho / a.group, h = sp.kvh * a.group + rho - i * a.group;
    float x[NC][8];
#pragma unroll
    for (int c = 0; c < NC / 2; c++)
        q_values8<HD>(a, (long)sp.s * a.max_tok + i, h, 32 * c + 8 * g, pos, x[c], x[c + NC / 2]);
    constexpr float kRoot = HD == 64 ? 8.f : HD == 256 ? 16.f : 11.3137084989847603904f;
    scale = kLog2e / kRoot;
    float up = 1.f;
    if (Parts<T>::kScaleQ) {
        float top = 0.f;
#pragma unroll
        for (int c = 0; c < NC; c++)
#pragma unroll
            for (int e = 0; e < 8; e++) top = fmaxf(top, fabsf(x[c][e]));
        top = rows_max(top);
        // 2^(15 - exponent): the largest value between 2^14 and 2^15
        const int ex = top > 0.f ? min(max(15 - (int)__builtin_amdgcn_frexp_expf(top), -100), 100) : 0;
        up = __builtin_ldexpf(1.f, ex);
        scale = __builtin_ldexpf(scale, -ex);
    } else {
        float high = 0.f;
        uint32_t low = ~0u;
#pragma unroll
        for (int c = 0; c < NC; c++)
#pragma unroll
            for (int e = 0; e < 8; e++) {
                high = fmaxf(high, fabsf(x[c][e]));
                low = min(low, (__float_as_uint(x[c][e]) & 0x7fffffffu) - 1u);
            }
        // NaN of one lane reaches O and the weights' sum from its keys
        scale = q_splits(high, low) ? scale : NAN;
    }
#pragma unroll
    for (int c = 0; c < NC; c++) {
#pragma unroll
        for (int e = 0; e < 8; e++) x[c][e] *= up;
        Parts<T>::split_q(x[c], qf[c]);
    }
}

// The weights of one step for the lane's query row from S^T's two tiles: masks,
// running maximum and sum, and P as the second product's operand.  keep: what O is
// multiplied by.  bad: bit (4 tile + r) set where the lane's key is no row.
template <class T>
__device__ __forceinline__ void weights(const f32x4 (&st)[2][Parts<T>::SUMS], float scale, bool masked,
                                        uint64_t mask, int jb, const Span& sp, uint32_t bad, float& m,
                                        float& l, float& keep, uint4 (&pf)[Parts<T>::QP]) {
    const int g = (threadIdx.x & 63) >> 4;
    float s[8];
#pragma unroll
    for (int e = 0; e < 8; e++) s[e] = Parts<T>::total(st[e >> 2], e & 3);
    if (masked) {
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const int j = jb + 16 * (e >> 2) + 4 * g + (e & 3);
            // without branches; a key that the cache held is seen by all
            const uint32_t own = j >= sp.held ? (uint32_t)(mask >> ((j - sp.held) & 63)) : 1u;
            const uint32_t see = own & ~(bad >> e) & (uint32_t)(j < sp.j1);
            s[e] = see & 1 ? s[e] : -INFINITY;
        }
    }
    float top = s[0];
#pragma unroll
    for (int e = 1; e < 8; e++) top = fmaxf(top, s[e]);
    top = rows_max(top) * scale;
    const float mn = fmaxf(m, top);
    const float base = mn == -INFINITY ? 0.f : mn;
    keep = __builtin_amdgcn_exp2f(m - base);
    float p[8], sum = 0.f;
#pragma unroll
    for (int e = 0; e < 8; e++) {
        p[e] = __builtin_amdgcn_exp2f(fmaf(s[e], scale, -base));
        sum += p[e];
    }
    l = fmaf(l, keep, sum);
    m = mn;
    Parts<T>::split_p(p, pf);
}

// Shares that follow each other run on one XCD (workgroups go round the XCDs): their
// parts' row tiles, or beams' shared pages, are in one L2.
__device__ __forceinline__ int share_id() {
    const int n = gridDim.x;  // a multiple of 8
    return (blockIdx.x & 7) * (n >> 3) + (blockIdx.x >> 3);
}

// Row of out (of HD floats) that query row rho of a span is.
__device__ __forceinline__ long out_row(const PagedArgs& a, const Span& sp, int rho) {
    const int G = a.group;
    return ((long)sp.s * a.max_tok + rho / G) * a.n_heads + sp.kvh * G + rho % G;
}

// The shares' loop of both kernels: `body` for each stretch of this workgroup's share.
template <class Body>
__device__ __forceinline__ void for_spans(const PagedArgs& a, int tile_rows, Body body) {
    __shared__ long cum[kPlanSeqs + 1], scan[4];
    __shared__ SeqLen lens[kPlanSeqs];
    make_plan(a, tile_rows, cum, scan, lens);
    if (blockIdx.x == 0)
        for (int s = threadIdx.x; s <= a.n_seq; s += blockDim.x) a.plan[s] = cum[s];
    const long all = uniform(cum[a.n_seq]);
    const int share = share_id(), used = shares_used(a, all);
    if (share >= used) return;
    long lo = uniform(share_start(all, share, used));
    const long hi = uniform(share_start(all, share + 1, used));
    int seq = 0;
    while (lo < hi) body(next_span(a, cum, lens, tile_rows, share, seq, lo, hi));
}

// ---- up to 16 query rows: a wave needs every K and V value once, so it loads them
// from memory straight into the operands' layout (K: lane's key row, 8 elements a chunk;
// V: 8 keys of HD/16 consecutive elements), no LDS in between.  The workgroup's four
// waves take every fourth step of the split and join at its end.
//
// Bound by HBM where the cache is long: 16 sequences of 4000 rows, 32/8 heads of 128, one
// token: F32 (525 MB) 96.6 us, 5.4 TB/s; F16 56.5 us, 4.6 TB/s (half the bytes for the same
// steps); 256 elements, 16/4 heads, F32 120 us, 4.4 TB/s (48 registers spilt, 188 bytes a
// lane).  One token @1024 (24 workgroups) is a chain of latencies, 11.9 us + 4.3 of the
// join: 1.6 to start, 1 for the lengths' plan, 1.2 for the span, 2.6 and 1.9 for the table's
// and then K's and q's loads, 3.1 for the step's arithmetic (splits, products and softmax of
// one wave a SIMD), 1.1 to join the waves.
constexpr int kFewWaves = 4;

template <int HD, class T>
__device__ __forceinline__ void few_span(const PagedArgs& a, const Span& sp) {
    constexpr int NC = HD / 32, ND = HD / 16, KP = Parts<T>::KP, QP = Parts<T>::QP,
                  SUMS = Parts<T>::SUMS;
    __shared__ float os[kFewWaves][16][HD + 4];
    __shared__ float ms[kFewWaves][16], ls[kFewWaves][16];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int n = lane & 15, g = lane >> 4, G = a.group;
    const int kvh = sp.kvh, tile = sp.tile, rows = sp.rows;
    const int rho = tile * 16 + n;
    const bool live = rho < rows;
    const long ld = (long)a.n_kv_heads * HD;
    const T* kb = static_cast<const T*>(a.k) + kvh * HD + 8 * g;
    const T* vb = static_cast<const T*>(a.v) + kvh * HD + n * ND;

    // table entries of the lane's K key of each tile, kept as they are until their rows
    // are asked for (arithmetic on them would wait for every load before theirs), and
    // those rows, -1: none
    auto pages_of = [&](int jb, int (&pg)[2]) {
#pragma unroll
        for (int t = 0; t < 2; t++)
            pg[t] = kv_page(min(jb + 16 * t + n, sp.j1 - 1), sp.table, a.table_ld, a.page_shift);
    };
    auto rows_of = [&](int jb, const int (&pg)[2], int (&r)[2]) {
#pragma unroll
        for (int t = 0; t < 2; t++)
            r[t] = (int)kv_row_of(min(jb + 16 * t + n, sp.j1 - 1), pg[t], a.table_ld, a.n_pages,
                                  a.page_shift);
    };
    T kr[2][NC][8], vr[2][4][ND];
    auto load_k = [&](const int (&r)[2]) {
#pragma unroll
        for (int t = 0; t < 2; t++) {
            const T* p = kb + (long)max(r[t], 0) * ld;
#pragma unroll
            for (int c2 = 0; c2 < NC; c2++)
                __builtin_memcpy(kr[t][c2], __builtin_assume_aligned(p + 32 * c2, 16), 8 * sizeof(T));
        }
    };
    auto load_v = [&](const int (&r)[2]) {
#pragma unroll
        for (int t = 0; t < 2; t++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int row = __shfl(r[t], 4 * g + e, 64);
                const T* p = vb + (long)max(row, 0) * ld;
                __builtin_memcpy(vr[t][e], __builtin_assume_aligned(p, ND * sizeof(T) < 16 ? 8 : 16),
                                 ND * sizeof(T));
            }
    };
    const int first = sp.j0 + wave * kStep, hop = kFewWaves * kStep;
    int r[2], rn[2], pg[2];
    const int rq = live ? rho : 0, iq = rq / G;
    const long rowq = (long)sp.s * a.max_tok + iq;
    pages_of(min(first, sp.j1 - 1), pg);
    const long pos = q_pos(a, rowq);
    const uint64_t mask = seen_mask(a, rowq, iq);
    if (first < sp.j1) {
        rows_of(first, pg, r);
        load_k(r);
        load_v(r);
        pages_of(first + hop, pg);
    }
    uint4 qf[NC][QP];
    float scale;
    load_q<HD, T>(a, sp, rq, pos, qf, scale);
    f32x4 o[ND];
#pragma unroll
    for (int d = 0; d < ND; d++) o[d] = f32x4{0.f, 0.f, 0.f, 0.f};
    float m = -INFINITY, l = 0.f;
    for (int jb = first; jb < sp.j1; jb += hop) {
        const bool more = jb + hop < sp.j1;
        f32x4 st[2][SUMS];
#pragma unroll
        for (int t = 0; t < 2; t++)
#pragma unroll
            for (int e = 0; e < SUMS; e++) st[t][e] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c2 = 0; c2 < NC; c2++) {
            uint4 kf[2][KP];
#pragma unroll
            for (int t = 0; t < 2; t++) {
                if constexpr (KP == 1)
                    __builtin_memcpy(&kf[t][0], kr[t][c2], 16);
                else
                    Parts<T>::split_kv(kr[t][c2], kf[t]);
            }
            const uint4* const qc[1] = {qf[c2]};
            f32x4* const to[2][1] = {{st[0]}, {st[1]}};
            Parts<T>::template scores<2, 1>(kf, qc, to);
        }
        // no row behind a key: only bad tables have such keys before j1
        const bool hole = __any(r[0] < 0 || r[1] < 0);
        uint32_t bad = 0;
        if (hole) {
#pragma unroll
            for (int e = 0; e < 8; e++)
                bad |= (uint32_t)(__shfl(r[e >> 2], 4 * g + (e & 3), 64) < 0) << e;
        }
        if (more) {
            rows_of(jb + hop, pg, rn);
            load_k(rn);
        }
        float keep;
        uint4 pf[QP];
        weights<T>(st, scale, hole || jb + kStep > min(sp.held, sp.j1), mask, jb, sp, bad, m, l, keep, pf);
#pragma unroll
        for (int d = 0; d < ND; d += 2) {
            uint4 vf[2][KP];
#pragma unroll
            for (int i = 0; i < 2; i++) {
                o[d + i] *= keep;
                T w[8];
#pragma unroll
                for (int e = 0; e < 8; e++) w[e] = vr[e >> 2][e & 3][d + i];
                if constexpr (KP == 1)
                    __builtin_memcpy(&vf[i][0], w, 16);
                else
                    Parts<T>::split_kv(w, vf[i]);
            }
            const uint4* const p[1] = {pf};
            f32x4* const to[2][1] = {{&o[d]}, {&o[d + 1]}};
            Parts<T>::template product<2, 1>(vf, p, to);
        }
        if (more) {
            load_v(rn);
            r[0] = rn[0];
            r[1] = rn[1];
            pages_of(jb + 2 * hop, pg);
        }
    }
    // the wave's sums, element (4 g + e) * ND + d of row n
    l = rows_sum(l);
#pragma unroll
    for (int d = 0; d < ND; d++)
#pragma unroll
        for (int e = 0; e < 4; e++)
            os[wave][n][(4 * g + e) * ND + d] = o[d][e] * (1.f / Parts<T>::kUp);
    if (g == 0) {
        ms[wave][n] = m;
        ls[wave][n] = l;
    }
    __syncthreads();
    // thread: row threadIdx.x / 16, every 16th float4 of it
    const int t = threadIdx.x >> 4, u = threadIdx.x & 15;
    if (tile * 16 + t < rows) {
        float top = ms[0][t];
#pragma unroll
        for (int w = 1; w < kFewWaves; w++) top = fmaxf(top, ms[w][t]);
        const float base = top == -INFINITY ? 0.f : top;
        float f[kFewWaves], sum = 0.f;
#pragma unroll
        for (int w = 0; w < kFewWaves; w++) {
            // a wave without a weight has nothing to add, whatever it holds
            f[w] = ls[w][t] == 0.f ? 0.f : __builtin_amdgcn_exp2f(ms[w][t] - base);
            sum = fmaf(ls[w][t], f[w], sum);
        }
        const bool whole = sp.slot < 0;
        float* dst;
        if (whole) {
            dst = a.out + out_row(a, sp, tile * 16 + t) * HD;
        } else {
            dst = a.part + ((long)sp.slot * 16 + t) * HD;
            if (u == 0) a.part_ml[sp.slot * 16 + t] = make_float2(top, sum);
        }
        const float by = !whole ? 1.f : far_out(top) ? NAN : (sum == 0.f ? 0.f : 1.f / sum);
        for (int d = 4 * u; d < HD; d += 64) {
            float y[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int w = 0; w < kFewWaves; w++) {
                if (ls[w][t] == 0.f) continue;
#pragma unroll
                for (int e = 0; e < 4; e++) y[e] = fmaf(os[w][t][d + e], f[w], y[e]);
            }
#pragma unroll
            for (int e = 0; e < 4; e++) dst[d + e] = y[e] * by;
        }
    }
    __syncthreads();
}

template <int HD, class T>
__global__ __launch_bounds__(64 * kFewWaves) void k_attn_paged_few(PagedArgs a) {
    for_spans(a, 16, [&](const Span& sp) { few_span<HD, T>(a, sp); });
}

// ---- more rows: the workgroup's NW waves share each step's K and V through LDS,
// split into operands once (by the thread that loaded them) and laid out as the
// operands' fragments (64 lanes x 16 bytes), so every LDS access is 1 KiB in a row.
// Wave w has the 16-row tiles w and w + NW (MW = 2) of the workgroup's 16 NW MW rows; a
// fragment read from LDS then feeds two tiles' products.  What a row tile costs
// beside its products is the cache read again, so a tile is as large as registers allow:
// 64 rows of 4 waves, two workgroups a CU, else 128 or 256 of 8 waves.  The next step's
// values are in flight while this one is multiplied.
//
// 16 trees of up to 48 tokens, 32/8 heads of 128 @8191, F32: 360 to 375 us called in a row,
// 375 to 488 (median 446, at some 1.7 GHz) launched one by one under the profiler; 243 us is
// what six bf16 products a value take at a large library product's rate.  No one unit bounds
// it: vector units busy 45%, matrix units 37%, waves waiting 31% of the time.  Of 402 us
// before its last steps, with half the products 307, without the splitting 371, with a third
// of the LDS reads 375, without loads 360, loads and splitting alone 231.  The two waves of
// a SIMD go through the step's phases together, between the same barriers.  F16 pages, 28/4
// heads, 48 tokens @8000: 128 elements 306 us (vector units 50%, matrix units 24%, waiting
// 36%), 64 elements 275 us (41%, 12%, 46%; 11.6 vector instructions a product: softmax and
// the splitting of p).  256 elements, F32, 16/4 heads, 48 tokens @4000: 464 us (24%, 23%,
// 62%; 50 registers spilt, 188 bytes a lane).  Tried: K of the next step multiplied under this one's
// softmax (427), one LDS buffer and 2 workgroups (419), raised priority around the
// products (400), 4 waves of three tiles (158 registers spilt, 822).

// LDS of one step's fragments, and how many steps' fit beside each other (two: one
// barrier a step instead of two) with the workgroups a CU is to hold.
template <int HD, class T>
constexpr int many_bytes() {
    return (2 * (HD / 32) + HD / 16) * Parts<T>::KP * 1024;
}
template <int HD, class T, int NW>
constexpr int many_bufs() {
    return 2 * many_bytes<HD, T>() <= (NW == 8 ? 144 : 72) * 1024 ? 2 : 1;
}

template <int HD, class T, int NW, int MW>
__device__ __forceinline__ void many_span(const PagedArgs& a, const Span& sp) {
    constexpr int NC = HD / 32, ND = HD / 16, KP = Parts<T>::KP, QP = Parts<T>::QP,
                  SUMS = Parts<T>::SUMS, TR = 16 * NW * MW, NB = many_bufs<HD, T, NW>();
    // a thread's part of a step: EK times 8 elements of a key's K; EV elements of 8 keys' V.
    // 8 waves have both to do only from 128 elements a head up: at 64 the first four
    // take K and the others V.
    constexpr bool kHalves = HD == 64 && NW == 8;
    constexpr int EK = kHalves ? 1 : 4 * HD / (64 * NW), EV = kHalves ? 1 : HD / 64 * 4 / NW;
    constexpr int VL = 2 * NC * KP * 64;  // V's fragments behind K's
    __shared__ uint4 frag[NB][VL + ND * KP * 64];
    __shared__ uint64_t masks[TR];
    __shared__ uint32_t holes[NB];  // byte g, bit 4 tile + r: key 16 tile + 4 g + r is no row
    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int n = lane & 15, g = lane >> 4, G = a.group;
    const int kvh = sp.kvh, rows = sp.rows, row0 = sp.tile * TR;
    const long ld = (long)a.n_kv_heads * HD;

    const bool do_k = !kHalves || wave < 4, do_v = !kHalves || wave >= 4;
    const int kt = t & 255;  // with kHalves; else t
    const int vg = wave & 3, vd = kHalves ? lane : (wave >> 2) * (64 * EV) + lane * EV;
    T kr[EK][8], vr[8][EV];
    int pg[2];  // table entries of keys t & 15 of both tiles (as in k_attn_paged_few)
    auto pages_of = [&](int jb) {
#pragma unroll
        for (int tt = 0; tt < 2; tt++)
            pg[tt] = kv_page(min(jb + 16 * tt + n, sp.j1 - 1), sp.table, a.table_ld, a.page_shift);
    };
    uint32_t bad_next = 0;
    // K unit p of the thread: key n of tile tt, elements 8 j ..
    auto k_unit = [&](int p, int& tt, int& j) {
        const int u = ((kHalves ? kt : t) >> 4) + 4 * NW * p;
        tt = u / (HD / 8);
        j = u % (HD / 8);
    };
    auto fetch = [&](int jb) {
        int krow[2], vrow[8];
#pragma unroll
        for (int tt = 0; tt < 2; tt++)
            krow[tt] = (int)kv_row_of(min(jb + 16 * tt + n, sp.j1 - 1), pg[tt], a.table_ld, a.n_pages,
                                      a.page_shift);
#pragma unroll
        for (int e = 0; e < 8; e++)
            vrow[e] = __builtin_amdgcn_readlane(krow[e >> 2], 4 * vg + (e & 3));
        // K: an address a lane; V: a scalar address a row and the lane's offset
        const T* kb = static_cast<const T*>(a.k) + kvh * HD;
        const T* vb = static_cast<const T*>(a.v) + kvh * HD;
        if (do_k) {
#pragma unroll
            for (int p = 0; p < EK; p++) {
                int tt, j;
                k_unit(p, tt, j);
                const size_t at = (size_t)max(tt ? krow[1] : krow[0], 0) * (size_t)ld + 8 * j;
                __builtin_memcpy(kr[p], __builtin_assume_aligned(kb + at, 16), 8 * sizeof(T));
            }
        }
        bad_next = 0;
#pragma unroll
        for (int e = 0; e < 8; e++) bad_next |= (uint32_t)(vrow[e] < 0) << e;
        if (do_v) {
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const T* row = vb + (size_t)max(vrow[e], 0) * (size_t)ld;
                __builtin_memcpy(vr[e], __builtin_assume_aligned(row + (uint32_t)vd, EV * sizeof(T)),
                                 EV * sizeof(T));
            }
        }
    };
    auto put = [&](int buf) {  // split what was fetched into LDS
        if (do_k) {
#pragma unroll
            for (int p = 0; p < EK; p++) {
                int tt, j;
                k_unit(p, tt, j);
                uint4 f[KP];
                if constexpr (KP == 1)
                    __builtin_memcpy(&f[0], kr[p], 16);
                else
                    Parts<T>::split_kv(kr[p], f);
#pragma unroll
                for (int q = 0; q < KP; q++)
                    frag[buf][((tt * NC + j / 4) * KP + q) * 64 + (j & 3) * 16 + n] = f[q];
            }
        }
        if (do_v) {
#pragma unroll
            for (int e = 0; e < EV; e++) {
                const int d = vd + e;
                T w[8];
#pragma unroll
                for (int r = 0; r < 8; r++) w[r] = vr[r][e];
                uint4 f[KP];
                if constexpr (KP == 1)
                    __builtin_memcpy(&f[0], w, 16);
                else
                    Parts<T>::split_kv(w, f);
#pragma unroll
                for (int q = 0; q < KP; q++)
                    frag[buf][VL + ((d >> 4) * KP + q) * 64 + vg * 16 + (d & 15)] = f[q];
            }
        }
        if (lane == 0 && wave < 4) reinterpret_cast<uint8_t*>(&holes[buf])[wave] = (uint8_t)bad_next;
    };

    pages_of(sp.j0);
    fetch(sp.j0);
    pages_of(sp.j0 + kStep);

    for (int r = t; r < TR; r += 64 * NW) {
        const int i = (row0 + r) / G;
        masks[r] = row0 + r < rows ? seen_mask(a, (long)sp.s * a.max_tok + i, i) : 0;
    }
    uint4 qf[MW][NC][QP];
    float scale[MW], m[MW], l[MW];
    bool act[MW];
    f32x4 o[MW][ND];
#pragma unroll
    for (int w = 0; w < MW; w++) {
        const int rho = row0 + (wave + NW * w) * 16 + n;
        act[w] = row0 + (wave + NW * w) * 16 < rows;
        const int rq = rho < rows ? rho : 0;
        load_q<HD, T>(a, sp, rq, q_pos(a, (long)sp.s * a.max_tok + rq / G), qf[w], scale[w]);
        m[w] = -INFINITY;
        l[w] = 0.f;
#pragma unroll
        for (int d = 0; d < ND; d++) o[w][d] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    put(0);
    if (sp.j0 + kStep < sp.j1) {
        fetch(sp.j0 + kStep);
        pages_of(sp.j0 + 2 * kStep);
    }
    int buf = 0;
    for (int jb = sp.j0; jb < sp.j1; jb += kStep) {
        __syncthreads();
        // M row tiles' products side by side; with one, two key tiles' or elements' tiles
        auto multiply = [&](auto tiles_of_wave) {
            constexpr int M = decltype(tiles_of_wave)::value, NA = 3 - M;
            f32x4 st[M][2][SUMS];
#pragma unroll
            for (int w = 0; w < M; w++)
#pragma unroll
                for (int tt = 0; tt < 2; tt++)
#pragma unroll
                    for (int e = 0; e < SUMS; e++) st[w][tt][e] = f32x4{0.f, 0.f, 0.f, 0.f};
            // fragments are read one product ahead of their use, before that one's operands
            // are waited for, and no further: the scheduling barriers (more of them in
            // flight would not fit in registers)
            uint4 f[2][NA][KP];
            auto read_k = [&](int i) {  // product i: chunk i / (2 / NA), key tiles from i % (2 / NA) * NA
#pragma unroll
                for (int x = 0; x < NA; x++)
#pragma unroll
                    for (int p = 0; p < KP; p++)
                        f[i & 1][x][p] =
                            frag[buf][(((i % (2 / NA) * NA + x) * NC + i / (2 / NA)) * KP + p) * 64 + lane];
            };
            read_k(0);
#pragma unroll
            for (int i = 0; i < 2 * NC / NA; i++) {
                if (i + 1 < 2 * NC / NA) read_k(i + 1);
                __builtin_amdgcn_sched_barrier(0);
                const uint4* q[M];
                f32x4* to[NA][M];
#pragma unroll
                for (int w = 0; w < M; w++) {
                    q[w] = qf[w][i / (2 / NA)];
#pragma unroll
                    for (int x = 0; x < NA; x++) to[x][w] = st[w][i % (2 / NA) * NA + x];
                }
                Parts<T>::template scores<NA, M>(f[i & 1], q, to);
                __builtin_amdgcn_sched_barrier(0);
            }
            const uint32_t hole = holes[buf], bad = (hole >> (8 * g)) & 255;
            uint4 pf[M][QP];
            const uint4* p[M];
#pragma unroll
            for (int w = 0; w < M; w++) {
                float keep;
                const bool masked = hole || jb + kStep > min(sp.held, sp.j1);
                const uint64_t mask = masked ? masks[(wave + NW * w) * 16 + n] : 0;
                weights<T>(st[w], scale[w], masked, mask, jb, sp, bad, m[w], l[w], keep, pf[w]);
                p[w] = pf[w];
                if (__any(keep != 1.f)) {  // seldom after the first steps
#pragma unroll
                    for (int d = 0; d < ND; d++) o[w][d] *= keep;
                }
            }
            auto read_v = [&](int i) {
#pragma unroll
                for (int x = 0; x < NA; x++)
#pragma unroll
                    for (int q = 0; q < KP; q++)
                        f[i & 1][x][q] = frag[buf][VL + ((i * NA + x) * KP + q) * 64 + lane];
            };
            __builtin_amdgcn_sched_barrier(0);
            read_v(0);
#pragma unroll
            for (int i = 0; i < ND / NA; i++) {
                if (i + 1 < ND / NA) read_v(i + 1);
                __builtin_amdgcn_sched_barrier(0);
                f32x4* to[NA][M];
#pragma unroll
                for (int x = 0; x < NA; x++)
#pragma unroll
                    for (int w = 0; w < M; w++) to[x][w] = &o[w][i * NA + x];
                Parts<T>::template product<NA, M>(f[i & 1], p, to);
                __builtin_amdgcn_sched_barrier(0);
            }
        };
        if (MW == 2 && act[MW - 1])
            multiply(std::integral_constant<int, MW>());
        else if (act[0])
            multiply(std::integral_constant<int, 1>());
        if (NB == 1) __syncthreads();
        if (jb + kStep < sp.j1) {
            buf = NB == 1 ? 0 : buf ^ 1;
            put(buf);
            if (jb + 2 * kStep < sp.j1) {
                fetch(jb + 2 * kStep);
                pages_of(jb + 3 * kStep);
            }
        }
    }
    __syncthreads();
    const bool whole = sp.slot < 0;
#pragma unroll
    for (int w = 0; w < MW; w++) {
        if (!act[w]) continue;
        l[w] = rows_sum(l[w]);
        const int in = (wave + NW * w) * 16;  // the tile's first row within the workgroup's
        if (row0 + in + n >= rows) continue;
        float* dst = whole ? a.out + out_row(a, sp, row0 + in + n) * HD
                           : a.part + ((long)sp.slot * TR + in + n) * HD;
        if (!whole && g == 0) a.part_ml[sp.slot * TR + in + n] = make_float2(m[w], l[w]);
        const float by =
            (!whole ? 1.f : far_out(m[w]) ? NAN : (l[w] == 0.f ? 0.f : 1.f / l[w])) / Parts<T>::kUp;
#pragma unroll
        for (int d = 0; d < ND; d++) {
            f32x4_a4 y;
#pragma unroll
            for (int e = 0; e < 4; e++) y[e] = o[w][d][e] * by;
            *reinterpret_cast<f32x4_a4*>(dst + 16 * d + 4 * g) = y;
        }
    }
}

template <int HD, class T, int NW, int MW>
__global__ __launch_bounds__(64 * NW, NW == 4 && HD == 256 && sizeof(T) == 4 ? 1 : 2)
void k_attn_paged_many(PagedArgs a) {
    for_spans(a, 16 * NW * MW, [&](const Span& sp) { many_span<HD, T, NW, MW>(a, sp); });
}

// One wave a query row and head.  Where its part lies in several shares, their sums are
// brought to one base and added in their order, and divided by the weights' sum (lane j
// has share j's m and l, so one load's latency covers 64 of them); a whole part's row
// is read back.  A row that is not finite is done again with care, and so is one of F32
// pages with an element so small that the three parts have lost its digits.  4.3 us for 16
// rows, 4.4 for 672 (launch and three loads after each other: plan, m and l, sums), 0.4 more
// with Q8_0 blocks for 512; 19.6 us for 24576 rows of 128 whose 256 shares' sums are 34 MB.
template <int HD, class T>
__global__ __launch_bounds__(256) void k_attn_paged_join(PagedArgs a, int tile_rows) {
    constexpr int E = HD / 64, U = 8;
    const int lane = threadIdx.x & 63;
    const uint32_t w = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6));
    if (w >= (uint32_t)a.n_seq * a.max_tok * a.n_heads) return;  // at most 2^26
    const uint32_t token = w / (uint32_t)a.n_heads;
    const int h = (int)(w - token * a.n_heads), s = (int)(token / (uint32_t)a.max_tok);
    const int i = (int)token - s * a.max_tok, G = a.group;
    const long all = a.plan[a.n_seq], before = a.plan[s];
    const SeqLen n = seq_len(a.len, a.n_tok, a.max_tok, s, a.table_ld, a.page_shift);
    if (i >= n.tok) return;
    const SeqWork sw = seq_work(n, G, tile_rows, a.per);
    const int kvh = (int)((uint32_t)h / (uint32_t)G), rho = i * G + h - kvh * G;
    const int tile = rho >> __builtin_ctz(tile_rows);
    const long p0 = before + kvh * sw.of_head() + tile * sw.units;
    const long p1 = p0 + (tile == sw.tiles - 1 ? sw.last : sw.units) - 1;
    const int shares = shares_used(a, all);
    const int w1 = __builtin_amdgcn_readfirstlane(share_of(all, p0, shares));
    const int w2 = __builtin_amdgcn_readfirstlane(share_of(all, p1, shares));
    float* dst = a.out + (long)w * HD + lane * E;
    float o[E], l = 1.f;
    if (w1 == w2) {
#pragma unroll
        for (int e = 0; e < E; e++) o[e] = dst[e];
    } else {
        const int at = rho & (tile_rows - 1), used = w2 - w1 + 1;
        // the part's first share has it last, the others first
        auto slot = [&](int j) { return (long)(j == 0 ? 2 * w1 + 1 : 2 * (w1 + j)) * tile_rows + at; };
        // the sums of shares j0 .. j0 + U - 1, on their way while the weights are found
        auto sums = [&](int j0, float (&v)[U][E]) {
#pragma unroll
            for (int j = 0; j < U; j++)
#pragma unroll
                for (int e = 0; e < E; e++)
                    v[j][e] = a.part[slot(min(j0 + j, used - 1)) * HD + lane * E + e];
        };
        float v[U][E];
        float2 ml = lane < used ? a.part_ml[slot(lane)] : make_float2(-INFINITY, 0.f);
        sums(0, v);
        float top = ml.x;
        for (int j = lane + 64; j < used; j += 64) top = fmaxf(top, a.part_ml[slot(j)].x);
        top = wave_max(top);
        const float base = top == -INFINITY ? 0.f : top;
        l = 0.f;
#pragma unroll
        for (int e = 0; e < E; e++) o[e] = 0.f;
        for (int b = 0; b < used; b += 64) {
            if (b) ml = b + lane < used ? a.part_ml[slot(b + lane)] : make_float2(-INFINITY, 0.f);
            const float f = ml.y == 0.f ? 0.f : __builtin_amdgcn_exp2f(ml.x - base);
            l += wave_sum(ml.y * f);
            const int here = min(64, used - b);
            for (int j0 = 0; j0 < here; j0 += U) {
                if (b + j0) sums(b + j0, v);
#pragma unroll
                for (int j = 0; j < U; j++) {
                    const float fj = j0 + j < here ? __uint_as_float(__builtin_amdgcn_readlane(
                                                         __float_as_uint(f), (j0 + j) & 63))
                                                   : 0.f;
                    if (fj == 0.f) continue;  // no weight there, whatever it holds
#pragma unroll
                    for (int e = 0; e < E; e++) o[e] = fmaf(v[j][e], fj, o[e]);
                }
            }
        }
        const float by = far_out(top) ? NAN : (l == 0.f ? 0.f : 1.f / l);
#pragma unroll
        for (int e = 0; e < E; e++) o[e] *= by;
    }
    float check = l * 0.f;
    bool small = false;
#pragma unroll
    for (int e = 0; e < E; e++) {
        check = fmaf(o[e], 0.f, check);
        if (sizeof(T) == 4) small |= fabsf(o[e]) < kSmall && o[e] != 0.f;
    }
    const bool again = __any(check != 0.f || small);
    if (again) row_careful<HD, T>(a, s, i, h, o);
    if (again || w1 != w2) {
#pragma unroll
        for (int e = 0; e < E; e++) dst[e] = o[e];
    }
    if (a.outq8) {
        // a block's 32 values are in 32 / E neighbouring lanes
        float amax = 0.f;
#pragma unroll
        for (int e = 0; e < E; e++) amax = fmaxf(amax, fabsf(o[e]));
#pragma unroll
        for (int off = 16 / E; off > 0; off >>= 1) amax = fmaxf(amax, __shfl_xor(amax, off, 64));
        const float id = amax > 0.f ? 127.f / amax : 0.f;
        uint8_t* blk = a.outq8 + ((long)w * (HD / 32) + lane * E / 32) * Q8_0_BYTES;
#pragma unroll
        for (int e = 0; e < E; e++) {
            const float r = fminf(fmaxf(rintf(o[e] * id), -128.f), 127.f);
            blk[4 + (lane * E + e) % 32] = (uint8_t)(__builtin_isinf(id) ? -128 : (int)r);
        }
        if ((lane * E) % 32 == 0) *reinterpret_cast<float*>(blk) = amax / 127.f;
    }
}

// ---- store -----------------------------------------------------------------
// One thread 4 + 4 values of K (a RoPE pair's halves) and of V: element d..d+3 and
// d+HD/2.. of one head.  Each value is read and written once: 24 sequences of 48 tokens,
// 8 heads of 128, F16 (14.1 MB) 4.1 us, 3.4 TB/s; 8 rows of 2 heads of 128 3.1 us, a
// launch's time.
template <int HD, class T>
__global__ __launch_bounds__(256) void k_kv_store(KvStoreArgs a) {
    constexpr int PER = HD / 8;  // threads a head
    const int per_row = a.n_kv_heads * PER;
    const long t = (long)blockIdx.x * 256 + threadIdx.x;
    const long row = div_whole(t, per_row);
    if (row >= (long)a.n_seq * a.max_tok) return;
    const int s = (int)((uint32_t)row / (uint32_t)a.max_tok), i = (int)row - s * a.max_tok;
    const SeqLen n = seq_len(a.len, a.n_tok, a.max_tok, s, a.table_ld, a.page_shift);
    if (i >= n.tok) return;
    const int u = (int)(t - row * per_row), h = u / PER, d = (u % PER) * 4;
    const int at = h * HD + d;
    // every load before the first use of one
    const int page = kv_page(n.held + i, a.table + (long)s * a.table_ld, a.table_ld, a.page_shift);
    const long p = a.pos ? min(max(a.pos[row], 0), a.n_pos - 1) : 0;
    auto ld4 = [](const float* q) { return *reinterpret_cast<const f32x4_a4*>(q); };
    f32x4_a4 x = ld4(a.xk + row * a.k_ld + at), y = ld4(a.xk + row * a.k_ld + at + HD / 2);
    f32x4_a4 z = ld4(a.xv + row * a.v_ld + at), w = ld4(a.xv + row * a.v_ld + at + HD / 2);
    if (a.bk) {
        x += ld4(a.bk + at);
        y += ld4(a.bk + at + HD / 2);
    }
    if (a.bv) {
        z += ld4(a.bv + at);
        w += ld4(a.bv + at + HD / 2);
    }
    if (a.pos) {
        const f32x4_a4 c = ld4(a.cos_t + p * (HD / 2) + d), sn = ld4(a.sin_t + p * (HD / 2) + d);
        const f32x4_a4 x0 = x;
        x = x0 * c - y * sn;
        y = y * c + x0 * sn;
    }
    const long r = kv_row_of(n.held + i, page, a.table_ld, a.n_pages, a.page_shift);
    if (r < 0) return;
    T* k = static_cast<T*>(a.k) + r * a.n_kv_heads * HD + at;
    T* v = static_cast<T*>(a.v) + r * a.n_kv_heads * HD + at;
    auto st4 = [](T* q, const f32x4_a4& f) {  // F16 pages: to nearest, ties to even
        T o[4];
#pragma unroll
        for (int e = 0; e < 4; e++) o[e] = (T)f[e];
        __builtin_memcpy(__builtin_assume_aligned(q, 4 * sizeof(T)), o, sizeof(o));
    };
    st4(k, x);
    st4(k + HD / 2, y);
    st4(v, z);
    st4(v + HD / 2, w);
}

// ---- fork --------------------------------------------------------------------
// The tables are small (some ten thousand entries), so one workgroup walks them with
// barriers between its steps and no other launch.  Reference counts are atomics (whole
// numbers, so their order does not matter), in LDS up to kForkLdsPages pages: one CU's
// scattered atomics to L2 go one a cycle or less, 128 sequences of 49 pages took 19 us
// with them.  Everything else goes by index order.  4 beams @1000 5.6 us, 16 x 8 @1500
// 8.7: the walk's steps after each other, each a load's or a scan's latency.  Past what LDS
// holds it is the atomics: 64 x 2 sequences @12000 in 48448 pages, 192000 entries, 326 us.
constexpr int kForkThreads = 1024;
constexpr int kForkLdsPages = 32768;  // 128 KiB

__device__ __forceinline__ int ld_dev(const int* p) {
    return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ void st_dev(int* p, int v) {
    __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// Exclusive prefix sum of v over the workgroup; *total: the sum.  red: 17 ints.
__device__ __forceinline__ int block_scan(int v, int* red, int* total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int x = v;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const int y = __shfl_up(x, off, 64);
        if (lane >= off) x += y;
    }
    if (lane == 63) red[wave] = x;
    __syncthreads();
    if (threadIdx.x == 0) {
        int sum = 0;
        for (int w = 0; w < kForkThreads / 64; w++) {
            const int c = red[w];
            red[w] = sum;
            sum += c;
        }
        red[kForkThreads / 64] = sum;
    }
    __syncthreads();
    const int before = red[wave] + x - v;
    *total = red[kForkThreads / 64];
    __syncthreads();
    return before;
}

// Output sequence i: what it keeps and where its room ends, in pages.
struct ForkSeq {
    int src;    // input row, or -1: holds nothing
    int full;   // pages shared
    int tail;   // rows of the page that has to be its own, 0: none
    int need;   // pages of rows and room
};
__device__ __forceinline__ ForkSeq fork_seq(const KvForkArgs& a, int i) {
    ForkSeq f = {-1, 0, 0, 0};
    const int s = a.parent[i], L = a.len[i];
    if (s < 0 || s >= a.n_in || L < 0) return f;
    const int n = kv_len(L, a.table_ld, a.page_shift), pr = 1 << a.page_shift;
    f.src = s;
    f.full = (a.extra > 0 ? n : n + pr - 1) >> a.page_shift;
    f.tail = a.extra > 0 ? n & (pr - 1) : 0;
    f.need = (int)min((long)a.table_ld, ((long)n + a.extra + pr - 1) >> a.page_shift);
    return f;
}

template <bool kLds>
__global__ __launch_bounds__(kForkThreads) void k_kv_fork(KvForkArgs a) {
    extern __shared__ int lds_refs[];
    __shared__ int red[kForkThreads / 64 + 1];
    __shared__ int src_of[kForkThreads], full_of[kForkThreads];  // of the first outputs
    __shared__ int copies;
    const int t = threadIdx.x;
    int* first = a.scratch;             // n_pages: lowest output that ends in the page
    int* free_list = first + a.n_pages;  // n_pages
    int* copy = free_list + a.n_pages;  // n_out x {source page, destination page, rows}
    if (t == 0) copies = 0;
    const ForkSeq mine = t < a.n_out ? fork_seq(a, t) : ForkSeq{-1, 0, 0, 0};
    src_of[t] = mine.src;
    full_of[t] = mine.full;
    auto seq_of = [&](int i) { return i == t ? mine : fork_seq(a, i); };
    auto add_ref = [&](int p, int v) { atomicAdd(kLds ? lds_refs + p : a.refs_out + p, v); };
    auto ref_of = [&](int p) { return kLds ? lds_refs[p] : ld_dev(a.refs_out + p); };
    if (kLds) {
        for (int p = t; p < a.n_pages; p += kForkThreads) lds_refs[p] = a.refs[p];
    } else if (a.refs_out != a.refs) {
        for (int p = t; p < a.n_pages; p += kForkThreads) st_dev(a.refs_out + p, a.refs[p]);
    }
    __syncthreads();
    // what the input rows hold is let go, what the outputs share is taken; U entries'
    // loads are in flight together
    constexpr int U = 4;
    const long n_old = (long)a.n_in * a.table_ld, n_new = (long)a.n_out * a.table_ld;
    for (long e0 = t; e0 < n_old; e0 += U * kForkThreads) {
        int p[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const long e = e0 + u * kForkThreads;
            p[u] = e < n_old ? a.table[e] : -1;
        }
#pragma unroll
        for (int u = 0; u < U; u++)
            if (p[u] >= 0 && p[u] < a.n_pages) add_ref(p[u], -1);
    }
    for (long e0 = t; e0 < n_new; e0 += U * kForkThreads) {
        int p[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const long e = e0 + u * kForkThreads;
            p[u] = -1;
            if (e >= n_new) continue;
            const int i = (int)div_whole(e, a.table_ld), col = (int)(e - (long)i * a.table_ld);
            int src, full;
            if (i < kForkThreads) {
                src = src_of[i];
                full = full_of[i];
            } else {
                const ForkSeq f = fork_seq(a, i);
                src = f.src;
                full = f.full;
            }
            if (col < full) p[u] = a.table[(long)src * a.table_ld + col];
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            const long e = e0 + u * kForkThreads;
            if (e >= n_new) continue;
            const bool page = p[u] >= 0 && p[u] < a.n_pages;
            if (page) add_ref(p[u], 1);
            a.table_out[e] = page ? p[u] : -1;
        }
    }
    // pages that an output ends in: the lowest output there may keep it
    for (int i = t; i < a.n_out; i += kForkThreads) {
        const ForkSeq f = seq_of(i);
        int p = -1;
        if (f.tail) {
            p = a.table[(long)f.src * a.table_ld + f.full];
            if (p < 0 || p >= a.n_pages) p = -1;
        }
        copy[3 * i] = p;
        if (p >= 0) st_dev(first + p, a.n_out);
    }
    __syncthreads();
    for (int i = t; i < a.n_out; i += kForkThreads)
        if (copy[3 * i] >= 0) atomicMin(first + copy[3 * i], i);
    __syncthreads();
    for (int i = t; i < a.n_out; i += kForkThreads) {
        const int p = copy[3 * i];
        copy[3 * i + 2] = p >= 0 && ld_dev(first + p) == i && ref_of(p) == 0;
    }
    __syncthreads();
    // the kept ones counted; each output's place among the pages to take
    int want = 0;
    for (int i0 = 0; i0 < a.n_out; i0 += kForkThreads) {
        const int i = i0 + t;
        int c = 0, keep = 0;
        if (i < a.n_out) {
            const ForkSeq f = seq_of(i);
            keep = copy[3 * i + 2];
            if (keep) {
                const int p = copy[3 * i];
                add_ref(p, 1);
                a.table_out[(long)i * a.table_ld + f.full] = p;
            }
            c = max(0, f.need - f.full - keep);
        }
        int sum;
        const int before = block_scan(c, red, &sum);
        if (i < a.n_out) {
            if (keep) copy[3 * i] = -1;
            copy[3 * i + 1] = want + before;
            copy[3 * i + 2] = keep;
        }
        want += sum;
    }
    __syncthreads();
    // the free pages in order, four a thread and round
    int n_free = 0;
    for (int p0 = 0; p0 < a.n_pages; p0 += 4 * kForkThreads) {
        const int p = p0 + 4 * t;
        int is[4];
#pragma unroll
        for (int u = 0; u < 4; u++) is[u] = p + u < a.n_pages ? ref_of(p + u) : 1;
        int mine_free = 0, sum;
#pragma unroll
        for (int u = 0; u < 4; u++) mine_free += is[u] == 0;
        int at = n_free + block_scan(mine_free, red, &sum);
#pragma unroll
        for (int u = 0; u < 4; u++)
            if (is[u] == 0) {
                if (at < want) free_list[at] = p + u;
                at++;
            }
        n_free += sum;
    }
    __syncthreads();
    for (int i = t; i < a.n_out; i += kForkThreads) {
        const ForkSeq f = seq_of(i);
        const int src = copy[3 * i], keep = copy[3 * i + 2];
        int at = copy[3 * i + 1], dst = -1;
        for (int col = f.full + keep; col < f.need; col++, at++) {
            const int p = at < n_free ? free_list[at] : -1;
            a.table_out[(long)i * a.table_ld + col] = p;
            if (p >= 0) add_ref(p, 1);  // nothing held it
            if (col == f.full) dst = p;
        }
        const bool copied = src >= 0 && dst >= 0;
        copy[3 * i] = copied ? src : -1;
        copy[3 * i + 1] = dst;
        copy[3 * i + 2] = f.tail;
        if (copied) atomicAdd(&copies, 1);
    }
    __syncthreads();
    if (kLds)
        for (int p = t; p < a.n_pages; p += kForkThreads) a.refs_out[p] = lds_refs[p];
    if (t == 0) {
        a.info[0] = copies;
        a.info[1] = max(0, want - n_free);
        a.info[2] = max(0, n_free - want);
    }
}

// The copied pages' rows: workgroup (output, layer and K or V, 16 KiB of the page).
// 128 pages' rows in 24 layers, 12.6 MB read and written again: 6.0 to 7.6 us, 3.3 to 4.2
// TB/s; 2.6 us where little is copied.
constexpr int kCopyBytes = 16384;

__global__ __launch_bounds__(256) void k_kv_copy(uint8_t* k, uint8_t* v, const int* copy,
                                                 long page_bytes, long row_bytes, int n_pages) {
    const int src = copy[3 * blockIdx.x], dst = copy[3 * blockIdx.x + 1];
    if (src < 0) return;
    const long bytes = copy[3 * blockIdx.x + 2] * row_bytes;
    const long at = (long)blockIdx.z * kCopyBytes;
    if (at >= bytes) return;
    const long end = min(bytes, at + kCopyBytes);
    uint8_t* pool = (blockIdx.y & 1 ? v : k) + (long)(blockIdx.y >> 1) * n_pages * page_bytes;
    const uint8_t* from = pool + src * page_bytes;
    uint8_t* to = pool + dst * page_bytes;
    for (long b = at + threadIdx.x * 16; b < end; b += 4096)
        *reinterpret_cast<uint4*>(to + b) = *reinterpret_cast<const uint4*>(from + b);
}

// ---- compaction -----------------------------------------------------------------
// Length of a path: it ascends, below 64.  A wave's lanes look at an entry each.
__device__ __forceinline__ int path_length(const int* way, int most) {
    const int lane = threadIdx.x & 63;
    const int v = lane < most ? way[lane] : -1, before = __shfl_up(v, 1, 64);
    const bool good = lane < most && v < 64 && v > (lane ? before : -1);
    const uint64_t bad = __ballot(!good);
    return bad ? __builtin_ctzll(bad) : 64;
}

// Workgroup (sequence, layer, K or V): each thread owns 16-byte columns and moves rows in
// path order, eight reads at a time.  path[i] >= i and ascending: a row is written
// only after every read of it (an earlier write goes to a lower row than every later read).
// 16 trees of 32 nodes in 32 layers of 4 KiB rows, 80 MB: 16 to 18.7 us (median 17.4, 4.6
// TB/s), near what a large copy reaches (5.2); one tree of 16 in 2 layers 2.9 us, a launch's
// time.
__global__ __launch_bounds__(256) void k_kv_compact(uint8_t* k, uint8_t* v, int* len_out,
                                                    const int* table, int table_ld,
                                                    const int* len, const int* path,
                                                    const int* n_path, int max_path, long row_bytes,
                                                    int n_pages, int page_shift, int write_len) {
    constexpr int U = 8;
    __shared__ int from[64], to[64];
    const int s = blockIdx.x, t = threadIdx.x;
    const int held = kv_len(len[s], table_ld, page_shift);
    const int* way = path + (long)s * max_path;
    const int n = path_length(way, min(max(n_path[s], 0), max_path));
    const int* row = table + (long)s * table_ld;
    if (t < n) {
        const int w = way[t];
        from[t] = (int)kv_row(held + w, row, table_ld, n_pages, page_shift);
        to[t] = w == t ? -1 : (int)kv_row(held + t, row, table_ld, n_pages, page_shift);
    }
    if (write_len && t == 0 && blockIdx.y == 0 && blockIdx.z == 0) len_out[s] = held + n;
    __syncthreads();
    uint8_t* pool = (blockIdx.z ? v : k) +
                    (((long)blockIdx.y * n_pages) << page_shift) * row_bytes;
    for (long b = t * 16; b < row_bytes; b += 4096) {
        for (int i0 = 0; i0 < n; i0 += U) {
            u32x4 x[U];  // read also where nothing moves: no branch between the reads
#pragma unroll
            for (int u = 0; u < U; u++)
                x[u] = *reinterpret_cast<const u32x4*>(
                    pool + (long)max(from[min(i0 + u, n - 1)], 0) * row_bytes + b);
#pragma unroll
            for (int u = 0; u < U; u++) {
                const int i = min(i0 + u, n - 1);
                if (i0 + u < n && from[i] >= 0 && to[i] >= 0)
                    *reinterpret_cast<u32x4*>(pool + (long)to[i] * row_bytes + b) = x[u];
            }
        }
    }
}

// len_out where it is len (or nothing moves): behind every workgroup that reads len.
__global__ __launch_bounds__(256) void k_kv_compact_len(int* len_out, const int* len,
                                                        const int* path, const int* n_path,
                                                        int n_seq, int max_path, int table_ld,
                                                        int page_shift) {
    const int s = blockIdx.x * 4 + (threadIdx.x >> 6);
    if (s >= n_seq) return;
    const int n = path_length(path + (long)s * max_path, min(max(n_path[s], 0), max_path));
    if ((threadIdx.x & 63) == 0) len_out[s] = kv_len(len[s], table_ld, page_shift) + n;
}

// Query rows of a KV head that a workgroup takes: the fewest that hold them all, up to
// 128.  Measured against the next larger tile: 16 sequences of 1000 to 4000 rows, 32/8 heads
// of 128, F32, one token (4 rows): 71.6 us, 64-row tiles 78.8; 12 tokens (48 rows): 93.3 us,
// 128-row tiles 103.6.  256 rows (two tiles a wave, each fragment read from LDS once for both; the
// cache read once for them, which L2 gives to 128-row tiles too) pay where the products are
// the least of a step, 64 elements a head with F16 pages: 16 trees of 48 tokens, 28/4
// heads, 2000 to 8000 rows: 169.7 us, 128-row tiles 184.1; F16 at 128 elements 191.7 and
// 190.0, F32 at 64 208.7 and 210.2; F32 at 128, 16 trees @8191 (40 registers spilt) 446 and
// 402.
int tile_rows(int rows, int head_dim, int kv_type) {
    if (rows <= 16) return 16;
    if (rows <= 64) return 64;
    return rows > 128 && head_dim == 64 && kv_type == AXF_TYPE_F16 ? 256 : 128;
}

template <int HD, class T>
hipError_t attn_launch(const PagedArgs& a, hipStream_t st) {
    const int tr = tile_rows(a.max_tok * a.group, HD,
                             sizeof(T) == 2 ? AXF_TYPE_F16 : AXF_TYPE_F32);
    if (tr == 16) {
        k_attn_paged_few<HD, T><<<a.shares, 64 * kFewWaves, 0, st>>>(a);
    } else if (tr == 64) {
        k_attn_paged_many<HD, T, 4, 1><<<a.shares, 256, 0, st>>>(a);
    } else if (tr == 128) {
        k_attn_paged_many<HD, T, 8, 1><<<a.shares, 512, 0, st>>>(a);
    } else {
        if constexpr (HD == 64 && sizeof(T) == 2)
            k_attn_paged_many<HD, T, 8, 2><<<a.shares, 512, 0, st>>>(a);
    }
    const long waves = (long)a.n_seq * a.max_tok * a.n_heads;
    k_attn_paged_join<HD, T><<<(unsigned)((waves + 3) / 4), 256, 0, st>>>(a, tr);
    return hipGetLastError();
}

hipError_t attn_types(const PagedArgs& a, int kv_type, int head_dim, hipStream_t st) {
    if (kv_type == AXF_TYPE_F16) {
        if (head_dim == 64) return attn_launch<64, _Float16>(a, st);
        if (head_dim == 128) return attn_launch<128, _Float16>(a, st);
        return attn_launch<256, _Float16>(a, st);
    }
    if (head_dim == 64) return attn_launch<64, float>(a, st);
    if (head_dim == 128) return attn_launch<128, float>(a, st);
    return attn_launch<256, float>(a, st);
}

template <int HD, class T>
hipError_t store_launch(const KvStoreArgs& a, hipStream_t st) {
    const long threads = (long)a.n_seq * a.max_tok * a.n_kv_heads * (HD / 8);
    k_kv_store<HD, T><<<(unsigned)((threads + 255) / 256), 256, 0, st>>>(a);
    return hipGetLastError();
}

}  // namespace

// Workgroups of the launch: as many as run at once, or as few as have a unit each by the
// caller's estimate of the lengths.  A CU holds two workgroups of 64-row tiles (with F32 at
// 256 elements one: LDS), or of few rows at 64 elements a head (fewer than 256 registers);
// one of few rows at 128 and 256 elements, or of 8 waves.  More than run at once leave the last
// ones a CU to themselves: 16 sequences of 1000 to 4000 rows, 32/8 heads, with 256, 512, 1024
// workgroups: 73, 83, 98 us; 12 tokens each, 16/4 heads of 256, F32 (96 KiB of LDS) with 256
// and 512: 134, 146.
void attn_paged_plan(PagedArgs& a, int kv_type, int head_dim, int max_len) {
    const long cap = (long)a.table_ld << a.page_shift;
    const long longest = (max_len < cap ? max_len : cap) + a.max_tok;
    const int rows = a.max_tok * a.group, tr = tile_rows(rows, head_dim, kv_type);
    const long seqs = a.n_seq < kPlanSeqs ? a.n_seq : kPlanSeqs;
    a.per = tr == 16 ? kFewWaves : (tr == 128 && rows > 128 ? 3 : 1);
    const long units = (longest + a.per * kStep - 1) / (a.per * kStep) * seqs * a.n_kv_heads *
                       ((rows + tr - 1) / tr);
    const bool alone = head_dim == 256 && kv_type == AXF_TYPE_F32;
    const long most = (tr == 64 && !alone) || (tr == 16 && head_dim == 64) ? 512 : 256;
    const long shares = units < most ? units : most;
    a.shares = (int)((shares + 7) & ~7L);
}

size_t attn_paged_scratch(const PagedArgs& a, int kv_type, int head_dim) {
    const int tr = tile_rows(a.max_tok * a.group, head_dim, kv_type);
    return (kPlanSeqs + 1) * sizeof(long) + (size_t)2 * a.shares * tr * (head_dim + 2) * 4 + 16;
}

hipError_t launch_attn_paged(const PagedArgs& a, int kv_type, int head_dim, void* scratch,
                             hipStream_t st) {
    const int tr = tile_rows(a.max_tok * a.group, head_dim, kv_type);
    for (int s = 0; s < a.n_seq; s += kPlanSeqs) {
        PagedArgs b = a;
        const long row = (long)s * a.max_tok;
        b.n_seq = a.n_seq - s < kPlanSeqs ? a.n_seq - s : kPlanSeqs;
        b.q += row * a.q_ld;
        b.table += (long)s * a.table_ld;
        b.len += s;
        if (b.n_tok) b.n_tok += s;
        if (b.mask) b.mask += row;
        if (b.pos) b.pos += row;
        b.out += row * a.n_heads * head_dim;
        if (b.outq8) b.outq8 += row * a.n_heads * (head_dim / 32) * Q8_0_BYTES;
        b.part = static_cast<float*>(scratch);
        b.part_ml = reinterpret_cast<float2*>(b.part + 2L * a.shares * tr * head_dim);
        b.plan = reinterpret_cast<long*>(b.part_ml + 2L * a.shares * tr);
        if (hipError_t e = attn_types(b, kv_type, head_dim, st); e != hipSuccess) return e;
    }
    return hipSuccess;
}

hipError_t launch_kv_store(const KvStoreArgs& a, int kv_type, int head_dim, hipStream_t st) {
    if (kv_type == AXF_TYPE_F16) {
        if (head_dim == 64) return store_launch<64, _Float16>(a, st);
        if (head_dim == 128) return store_launch<128, _Float16>(a, st);
        return store_launch<256, _Float16>(a, st);
    }
    if (head_dim == 64) return store_launch<64, float>(a, st);
    if (head_dim == 128) return store_launch<128, float>(a, st);
    return store_launch<256, float>(a, st);
}

size_t kv_fork_scratch(int n_pages, int n_out) {
    return ((size_t)n_pages * 2 + (size_t)n_out * 3 + 1) * 4;
}

hipError_t launch_kv_fork(const KvForkArgs& a, const axf_kv_pages& kv, hipStream_t st) {
    if (a.n_pages <= kForkLdsPages)
        k_kv_fork<true><<<1, kForkThreads, a.n_pages * sizeof(int), st>>>(a);
    else
        k_kv_fork<false><<<1, kForkThreads, 0, st>>>(a);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || a.extra == 0 || a.n_out == 0) return e;
    const long row_bytes = (long)kv.n_kv_heads * kv.head_dim * (kv.type == AXF_TYPE_F32 ? 4 : 2);
    const long page_bytes = row_bytes << a.page_shift;
    const dim3 grid(a.n_out, kv.n_layers * 2, (unsigned)((page_bytes + kCopyBytes - 1) / kCopyBytes));
    k_kv_copy<<<grid, 256, 0, st>>>(static_cast<uint8_t*>(kv.k), static_cast<uint8_t*>(kv.v),
                                    a.scratch + 2L * a.n_pages, page_bytes, row_bytes, kv.n_pages);
    return hipGetLastError();
}

hipError_t launch_kv_compact(const axf_kv_pages& kv, int* len_out, const int* table, int table_ld,
                             const int* len, const int* path, const int* n_path, int n_seq,
                             int max_path, hipStream_t st) {
    const int shift = __builtin_ctz((unsigned)kv.page_rows);
    const long row_bytes = (long)kv.n_kv_heads * kv.head_dim * (kv.type == AXF_TYPE_F32 ? 4 : 2);
    // len_out can be written by the workgroups that read len only where they are apart
    const bool apart = len_out + n_seq <= len || len + n_seq <= len_out;
    if (max_path > 0) {
        k_kv_compact<<<dim3(n_seq, kv.n_layers, 2), 256, 0, st>>>(
            static_cast<uint8_t*>(kv.k), static_cast<uint8_t*>(kv.v), len_out, table, table_ld, len,
            path, n_path, max_path, row_bytes, kv.n_pages, shift, apart);
        hipError_t e = hipGetLastError();
        if (e != hipSuccess || apart) return e;
    }
    k_kv_compact_len<<<(n_seq + 3) / 4, 256, 0, st>>>(len_out, len, path, n_path, n_seq, max_path,
                                                      table_ld, shift);
    return hipGetLastError();
}

}  // namespace axf
