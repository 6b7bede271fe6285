// paged.hip — a cache of K/V pages that several continuations of a text share:
// attention over it, the store of new rows, the fork of page tables, the
// compaction after a drafted tree was verified (include/axf_hip.h has the layout
// and the calls' rules).
#include "common.hpp"
#include "paged_index.hpp"

namespace axf {

namespace {

constexpr float kLog2e = 1.44269504088896340736f;

template <class T>
__device__ __forceinline__ float kv_value(T v) {
    return (float)v;
}

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

// ---- attention: one wave a query row ----------------------------------------
// Partial result of a split: m (the largest score * log2 e / sqrt(HD)), l (sum of
// 2^(score - m)) and o (the weighted V sum); the combine kernel joins them.
template <int HD, class T>
__global__ __launch_bounds__(256) void k_attn_paged_rows(PagedArgs a) {
    constexpr int E = HD / 64;
    const int lane = threadIdx.x & 63;
    const long w = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
    const long rows = (long)a.n_seq * a.max_tok * a.n_heads;
    if (w >= rows) return;
    const int h = (int)(w % a.n_heads);
    const long row = w / a.n_heads;
    const int i = (int)(row % a.max_tok), s = (int)(row / a.max_tok);
    const SeqLen n = seq_len(a.len, a.n_tok, a.max_tok, s, a.table_ld, a.page_shift);
    if (i >= n.tok) return;
    const int total = n.held + n.tok;
    const int j0 = blockIdx.y * a.split_rows;
    const int j1 = (int)blockIdx.y + 1 == a.nsplit ? total : min(total, j0 + a.split_rows);
    const int kvh = h / (a.n_heads / a.n_kv_heads);
    const int ld = a.n_kv_heads * HD;
    const uint64_t mask = a.mask ? a.mask[row] : ~0ull >> (63 - i);
    const int* table = a.table + (long)s * a.table_ld;
    const T* k = static_cast<const T*>(a.k) + kvh * HD;
    const T* v = static_cast<const T*>(a.v) + kvh * HD;
    const float c = kLog2e / sqrtf((float)HD);
    float q[E], o[E];
#pragma unroll
    for (int e = 0; e < E; e++) {
        q[e] = q_value<HD>(a, row, h, lane + 64 * e);
        o[e] = 0.f;
    }
    float m = -INFINITY, l = 0.f;
    for (int j = j0; j < j1; j++) {
        if (j >= n.held && !((mask >> (j - n.held)) & 1)) continue;
        const long r = kv_row(j, table, a.table_ld, a.n_pages, a.page_shift);
        if (r < 0) continue;
        float d = 0.f;
#pragma unroll
        for (int e = 0; e < E; e++) d = fmaf(q[e], kv_value(k[r * ld + lane + 64 * e]), d);
        d = wave_sum(d) * c;
        const float mn = fmaxf(m, d);
        const float base = mn == -INFINITY ? 0.f : mn;
        const float keep = exp2f(m - base), p = exp2f(d - base);
        l = l * keep + p;
#pragma unroll
        for (int e = 0; e < E; e++) o[e] = fmaf(p, kv_value(v[r * ld + lane + 64 * e]), o[e] * keep);
        m = mn;
    }
    if (a.nsplit == 1 && !a.outq8) {
        float* dst = a.out + row * a.n_heads * HD + h * HD;
#pragma unroll
        for (int e = 0; e < E; e++) dst[lane + 64 * e] = l == 0.f ? 0.f : o[e] / l;
        return;
    }
    float* dst = a.part + (w * a.nsplit + blockIdx.y) * (HD + 2);
    if (lane == 0) {
        dst[0] = m;
        dst[1] = l;
    }
#pragma unroll
    for (int e = 0; e < E; e++) dst[2 + lane + 64 * e] = o[e];
}

// One wave a query row and head: the splits' sums brought to one base and added
// in their order, divided by the weights' sum.
template <int HD>
__global__ __launch_bounds__(256) void k_attn_paged_join(PagedArgs a) {
    constexpr int E = HD / 64;
    const int lane = threadIdx.x & 63;
    const long w = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (w >= (long)a.n_seq * a.max_tok * a.n_heads) return;
    const int h = (int)(w % a.n_heads);
    const long row = w / a.n_heads;
    const int s = (int)(row / a.max_tok);
    const SeqLen n = seq_len(a.len, a.n_tok, a.max_tok, s, a.table_ld, a.page_shift);
    if ((int)(row % a.max_tok) >= n.tok) return;
    const int used = min(a.nsplit, (n.held + n.tok + a.split_rows - 1) / a.split_rows);
    const float* p = a.part + w * a.nsplit * (HD + 2);
    float top = -INFINITY;
    for (int j = 0; j < used; j++) top = fmaxf(top, p[(long)j * (HD + 2)]);
    const float base = top == -INFINITY ? 0.f : top;
    float l = 0.f, o[E];
#pragma unroll
    for (int e = 0; e < E; e++) o[e] = 0.f;
    for (int j = 0; j < used; j++) {
        const float* pj = p + (long)j * (HD + 2);
        const float f = exp2f(pj[0] - base);
        l = fmaf(pj[1], f, l);
#pragma unroll
        for (int e = 0; e < E; e++) o[e] = fmaf(pj[2 + lane + 64 * e], f, o[e]);
    }
    float* dst = a.out + row * a.n_heads * HD + h * HD;
#pragma unroll
    for (int e = 0; e < E; e++) {
        const float y = l == 0.f ? 0.f : o[e] / l;
        dst[lane + 64 * e] = y;
        if (a.outq8) {
            // lane & 31 of each half wave holds one block's values
            float amax = fabsf(y);
#pragma unroll
            for (int off = 16; off > 0; off >>= 1) amax = fmaxf(amax, __shfl_xor(amax, off, 64));
            const float id = amax > 0.f ? 127.f / amax : 0.f;
            const float r = fminf(fmaxf(rintf(y * id), -128.f), 127.f);
            const int b = __builtin_isinf(id) ? -128 : (int)r;
            uint8_t* blk = a.outq8 +
                           ((row * a.n_heads + h) * (HD / 32) + e * 2 + (lane >> 5)) * Q8_0_BYTES;
            blk[4 + (lane & 31)] = (uint8_t)b;
            if ((lane & 31) == 0) *reinterpret_cast<float*>(blk) = amax / 127.f;
        }
    }
}

// ---- store -----------------------------------------------------------------
// One thread 4 + 4 values of K (a RoPE pair's halves) and of V: element d..d+3 and
// d+HD/2.. of one head.  Bandwidth: each value is read and written once.
template <int HD, class T>
__global__ __launch_bounds__(256) void k_kv_store(KvStoreArgs a) {
    constexpr int PER = HD / 8;  // threads a head
    const int per_row = a.n_kv_heads * PER;
    const long t = (long)blockIdx.x * 256 + threadIdx.x;
    const long row = t / per_row;
    if (row >= (long)a.n_seq * a.max_tok) return;
    const int s = (int)(row / a.max_tok), i = (int)(row % a.max_tok);
    const SeqLen n = seq_len(a.len, a.n_tok, a.max_tok, s, a.table_ld, a.page_shift);
    if (i >= n.tok) return;
    const long r = kv_row(n.held + i, a.table + (long)s * a.table_ld, a.table_ld, a.n_pages,
                          a.page_shift);
    if (r < 0) return;
    const int u = (int)(t % per_row), h = u / PER, d = (u % PER) * 4;
    const int at = h * HD + d;
    T* k = static_cast<T*>(a.k) + r * a.n_kv_heads * HD + at;
    T* v = static_cast<T*>(a.v) + r * a.n_kv_heads * HD + at;
    const float* xk = a.xk + row * a.k_ld + at;
    const float* xv = a.xv + row * a.v_ld + at;
    const long p = a.pos ? min(max(a.pos[row], 0), a.n_pos - 1) : 0;
#pragma unroll
    for (int e = 0; e < 4; e++) {
        float x = xk[e], y = xk[e + HD / 2], z = xv[e], w = xv[e + HD / 2];
        if (a.bk) {
            x += a.bk[at + e];
            y += a.bk[at + e + HD / 2];
        }
        if (a.bv) {
            z += a.bv[at + e];
            w += a.bv[at + e + HD / 2];
        }
        if (a.pos) {
            const float c = a.cos_t[p * (HD / 2) + d + e], sn = a.sin_t[p * (HD / 2) + d + e];
            const float x0 = x;
            x = x0 * c - y * sn;
            y = y * c + x0 * sn;
        }
        // F16 pages: to nearest, ties to even
        k[e] = (T)x;
        k[e + HD / 2] = (T)y;
        v[e] = (T)z;
        v[e + HD / 2] = (T)w;
    }
}

// ---- fork --------------------------------------------------------------------
// The tables are small (some ten thousand entries), so one workgroup walks them with
// barriers between its steps and no other launch: reference counts as device-scope
// atomics (whole numbers, so their order does not matter), everything else by
// index order.
constexpr int kForkThreads = 1024;

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

__global__ __launch_bounds__(kForkThreads) void k_kv_fork(KvForkArgs a) {
    __shared__ int red[kForkThreads / 64 + 1];
    __shared__ int copies;
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    int* first = a.scratch;             // n_pages: lowest output that ends in the page
    int* free_list = first + a.n_pages;  // n_pages
    int* copy = free_list + a.n_pages;  // n_out x {source page, destination page, rows}
    if (t == 0) copies = 0;
    if (a.refs_out != a.refs)
        for (int p = t; p < a.n_pages; p += kForkThreads) st_dev(a.refs_out + p, a.refs[p]);
    __syncthreads();
    // what the input rows hold is let go, what the outputs share is taken
    for (long e = t; e < (long)a.n_in * a.table_ld; e += kForkThreads) {
        const int p = a.table[e];
        if (p >= 0 && p < a.n_pages) atomicAdd(a.refs_out + p, -1);
    }
    for (int i = wave; i < a.n_out; i += kForkThreads / 64) {
        const ForkSeq f = fork_seq(a, i);
        for (int col = lane; col < a.table_ld; col += 64) {
            int v = -1;
            if (col < f.full) {
                const int p = a.table[(long)f.src * a.table_ld + col];
                if (p >= 0 && p < a.n_pages) {
                    v = p;
                    atomicAdd(a.refs_out + p, 1);
                }
            }
            a.table_out[(long)i * a.table_ld + col] = v;
        }
    }
    // pages that an output ends in: the lowest output there may keep it
    for (int i = t; i < a.n_out; i += kForkThreads) {
        const ForkSeq f = fork_seq(a, i);
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
        copy[3 * i + 2] = p >= 0 && ld_dev(first + p) == i && ld_dev(a.refs_out + p) == 0;
    }
    __syncthreads();
    // the kept ones counted; each output's place among the pages to take
    int want = 0;
    for (int i0 = 0; i0 < a.n_out; i0 += kForkThreads) {
        const int i = i0 + t;
        int c = 0, keep = 0;
        if (i < a.n_out) {
            const ForkSeq f = fork_seq(a, i);
            keep = copy[3 * i + 2];
            if (keep) {
                const int p = copy[3 * i];
                atomicAdd(a.refs_out + p, 1);
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
    int n_free = 0;
    for (int p0 = 0; p0 < a.n_pages; p0 += kForkThreads) {
        const int p = p0 + t;
        const int is = p < a.n_pages && ld_dev(a.refs_out + p) == 0;
        int sum;
        const int at = n_free + block_scan(is, red, &sum);
        if (is && at < want) free_list[at] = p;
        n_free += sum;
    }
    __syncthreads();
    for (int i = t; i < a.n_out; i += kForkThreads) {
        const ForkSeq f = fork_seq(a, i);
        const int src = copy[3 * i], keep = copy[3 * i + 2];
        int at = copy[3 * i + 1], dst = -1;
        for (int col = f.full + keep; col < f.need; col++, at++) {
            const int p = at < n_free ? free_list[at] : -1;
            a.table_out[(long)i * a.table_ld + col] = p;
            if (p >= 0) st_dev(a.refs_out + p, 1);
            if (col == f.full) dst = p;
        }
        const bool copied = src >= 0 && dst >= 0;
        copy[3 * i] = copied ? src : -1;
        copy[3 * i + 1] = dst;
        copy[3 * i + 2] = f.tail;
        if (copied) atomicAdd(&copies, 1);
    }
    __syncthreads();
    if (t == 0) {
        a.info[0] = copies;
        a.info[1] = max(0, want - n_free);
        a.info[2] = max(0, n_free - want);
    }
}

// The copied pages' rows: workgroup (output, layer and K or V, 16 KiB of the page).
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
// Workgroup (sequence, layer, K or V): each thread owns 16-byte columns and
// moves rows in path order.  path[i] >= i and ascending, so no row is written before
// it was read.
__global__ __launch_bounds__(256) void k_kv_compact(uint8_t* k, uint8_t* v, int* len_out,
                                                    const int* table, int table_ld,
                                                    const int* len, const int* path,
                                                    const int* n_path, int max_path, long row_bytes,
                                                    int n_pages, int page_shift) {
    const int s = blockIdx.x;
    const int held = kv_len(len[s], table_ld, page_shift);
    const int* way = path + (long)s * max_path;
    const int most = min(max(n_path[s], 0), max_path);
    int n = 0;
    for (int last = -1; n < most && way[n] > last && way[n] < 64; n++) last = way[n];
    uint8_t* pool = (blockIdx.z ? v : k) +
                    (((long)blockIdx.y * n_pages) << page_shift) * row_bytes;
    const int* row = table + (long)s * table_ld;
    for (long b = threadIdx.x * 16; b < row_bytes; b += 4096) {
        for (int i = 0; i < n; i++) {
            if (way[i] == i) continue;
            const long from = kv_row(held + way[i], row, table_ld, n_pages, page_shift);
            const long to = kv_row(held + i, row, table_ld, n_pages, page_shift);
            if (from < 0 || to < 0) continue;
            *reinterpret_cast<uint4*>(pool + to * row_bytes + b) =
                *reinterpret_cast<const uint4*>(pool + from * row_bytes + b);
        }
    }
}

// len_out after the moves (it may be len): in a launch of its own, behind every
// workgroup that reads len.
__global__ __launch_bounds__(256) void k_kv_compact_len(int* len_out, const int* len,
                                                        const int* path, const int* n_path,
                                                        int n_seq, int max_path, int table_ld,
                                                        int page_shift) {
    const int s = blockIdx.x * 256 + threadIdx.x;
    if (s >= n_seq) return;
    const int* way = path + (long)s * max_path;
    const int most = min(max(n_path[s], 0), max_path);
    int n = 0;
    for (int last = -1; n < most && way[n] > last && way[n] < 64; n++) last = way[n];
    len_out[s] = kv_len(len[s], table_ld, page_shift) + n;
}

template <int HD, class T>
hipError_t attn_launch(const PagedArgs& a, hipStream_t st) {
    const long waves = (long)a.n_seq * a.max_tok * a.n_heads;
    const unsigned wgs = (unsigned)((waves + 3) / 4);
    k_attn_paged_rows<HD, T><<<dim3(wgs, a.nsplit), 256, 0, st>>>(a);
    if (a.nsplit > 1 || a.outq8) k_attn_paged_join<HD><<<wgs, 256, 0, st>>>(a);
    return hipGetLastError();
}

template <int HD, class T>
hipError_t store_launch(const KvStoreArgs& a, hipStream_t st) {
    const long threads = (long)a.n_seq * a.max_tok * a.n_kv_heads * (HD / 8);
    k_kv_store<HD, T><<<(unsigned)((threads + 255) / 256), 256, 0, st>>>(a);
    return hipGetLastError();
}

}  // namespace

void attn_paged_plan(PagedArgs& a, int kv_type, int head_dim, int max_len) {
    (void)kv_type;
    (void)head_dim;
    const long cap = (long)a.table_ld << a.page_shift;
    const long longest = (max_len < cap ? max_len : cap) + a.max_tok;
    const long waves = (long)a.n_seq * a.max_tok * a.n_heads;
    long split = longest * waves / 4096;
    split = split < 64 ? 64 : (split + 63) / 64 * 64;
    a.split_rows = (int)split;
    a.nsplit = (int)((longest + split - 1) / split);
}

size_t attn_paged_scratch(const PagedArgs& a, int head_dim) {
    if (a.nsplit == 1 && !a.outq8) return 0;
    return (size_t)a.n_seq * a.max_tok * a.n_heads * a.nsplit * (head_dim + 2) * 4;
}

hipError_t launch_attn_paged(const PagedArgs& a, int kv_type, int head_dim, hipStream_t st) {
    if (kv_type == AXF_TYPE_F16) {
        if (head_dim == 64) return attn_launch<64, _Float16>(a, st);
        if (head_dim == 128) return attn_launch<128, _Float16>(a, st);
        return attn_launch<256, _Float16>(a, st);
    }
    if (head_dim == 64) return attn_launch<64, float>(a, st);
    if (head_dim == 128) return attn_launch<128, float>(a, st);
    return attn_launch<256, float>(a, st);
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
    k_kv_fork<<<1, kForkThreads, 0, st>>>(a);
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
    if (max_path > 0) {
        k_kv_compact<<<dim3(n_seq, kv.n_layers, 2), 256, 0, st>>>(
            static_cast<uint8_t*>(kv.k), static_cast<uint8_t*>(kv.v), len_out, table, table_ld, len,
            path, n_path, max_path, row_bytes, kv.n_pages, shift);
        hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    k_kv_compact_len<<<(n_seq + 255) / 256, 256, 0, st>>>(len_out, len, path, n_path, n_seq, max_path,
                                                      table_ld, shift);
    return hipGetLastError();
}

}  // namespace axf
