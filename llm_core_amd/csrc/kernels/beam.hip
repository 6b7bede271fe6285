// beam.hip — beam search's selection: the best continuations of a sequence's beams
// over the vocabulary (axf_hip_beam_select).
//
//   score(b, t) = cum[b] + (x[b][t] - lse[b]),  lse[b] = log sum_t exp x[b][t]
//
// Which of two continuations is better may hang on the last bits of a score, so
// exponentials, sums and scores are 64-bit.  Within a beam the score rises with the
// logit, so one pass over the logits suffices:
//   1. k_beam_part: a workgroup takes a chunk of a row: its maximum m, sum of
//      exp(x - m) and its n_out largest (logit, lower token first) keys.
//   2. k_beam_merge: a workgroup a sequence joins the chunks' sums to each beam's
//      lse, turns the keys into scores and picks the n_out best of the chunks' sorted
//      lists.
// 8 x 8 beams of 151936 (38.9 MB, 7.5 us at a large copy's rate): 18.4 + 11.2 us (medians
// of a kernel trace).  The first: 38 vector instructions a logit, the 64-bit ones among
// them at half rate; the vector units are busy 63% of its time, the rest is ramp, loads and
// the 32 dependent ballots ahead of them (waves wait 44%).  The second: the latencies of one
// workgroup a sequence.  1 x 4 of 32000: 5.0 + 6.3 us.  A finished beam's row is read and
// summed like the others.
#include "common.hpp"

namespace axf {

namespace {

constexpr int kMergeThreads = 512;

__device__ __forceinline__ uint32_t ordered32(float v) {
    const uint32_t u = __float_as_uint(v + 0.f);  // -0 and +0 are one logit
    return u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
}
__device__ __forceinline__ float unordered32(uint32_t o) {
    return __uint_as_float((o & 0x80000000u) ? (o ^ 0x80000000u) : ~o);
}
__device__ __forceinline__ uint64_t ordered64(double v) {
    const uint64_t u = (uint64_t)__double_as_longlong(v + 0.0);
    return u ^ ((uint64_t)((int64_t)u >> 63) | 0x8000000000000000ull);
}
__device__ __forceinline__ double unordered64(uint64_t o) {
    return __longlong_as_double((int64_t)((o >> 63) ? (o ^ 0x8000000000000000ull) : ~o));
}

// 2^(j / 32), j < 32, to the nearest double: exp_neg's table, copied to LDS.
__device__ const double kExpTable[32] = {
    1.0, 1.0218971486541166,
    1.0442737824274138, 1.0671404006768237,
    1.0905077326652577, 1.1143867425958924,
    1.1387886347566916, 1.1637248587775775,
    1.189207115002721, 1.215247359980469,
    1.241857812073484, 1.2690509571917332,
    1.2968395546510096, 1.3252366431597413,
    1.3542555469368927, 1.383909881963832,
    1.4142135623730951, 1.4451808069770467,
    1.4768261459394993, 1.5091644275934228,
    1.5422108254079407, 1.5759808451078865,
    1.6104903319492543, 1.645755478153965,
    1.681792830507429, 1.718619298122478,
    1.7562521603732995, 1.7947090750031072,
    1.8340080864093424, 1.8741676341103,
    1.9152065613971474, 1.9571441241754002,
};
__device__ __forceinline__ void fill_exp_table(double* tab) {
    if (threadIdx.x < 32) tab[threadIdx.x] = kExpTable[threadIdx.x];
}

// exp(x) for x <= 0 to 3e-15 of its value near 0: 2^(k / 32) from the table times the Taylor
// polynomial of degree 5 on [-ln2/64, ln2/64] (its first term left out: 0.01083^6 / 6! =
// 2.2e-15), and to |x| 2^-54 more further out.  Below -708 zero; NaN stays NaN.
__device__ __forceinline__ double exp_neg(double x, const double* tab) {
    const double k = __builtin_rint(x * (32 * 1.4426950408889634074));
    // ln 2 / 32 in one part: off by 7.3e-19 a unit of k, 2.4e-14 at k = 32686
    const double r = __builtin_fma(k, -6.93147180559945309417e-01 / 32, x);
    double p = 1.0 / 120;
    p = __builtin_fma(p, r, 1.0 / 24);
    p = __builtin_fma(p, r, 1.0 / 6);
    p = __builtin_fma(p, r, 0.5);
    p = __builtin_fma(p, r, 1.0);
    const int n = (int)fmax(k, -32768.0);
    const double t = tab[n & 31];
    const double y = __builtin_ldexp(__builtin_fma(p * r, t, t), n >> 5);
    return x < -708.0 ? 0.0 : y;
}

__device__ __forceinline__ double wave_sum64(double v) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
    return v;
}

// The k-th largest of the wave's 64 values (k >= 1): bit by bit from the top, the
// largest value that at least k of them reach.
__device__ __forceinline__ uint32_t kth_of_wave(uint32_t v, int k) {
    uint32_t t = 0;
    for (int b = 31; b >= 0; b--) {
        const uint32_t c = t | (1u << b);
        if (__popcll(__ballot(v >= c)) >= k) t = c;
    }
    return t;
}

constexpr int kCap = 512;  // keys ranked at once

// Chunk blockIdx.x of row blockIdx.y: keys[n_out] (largest first, 0: none), m, s.
// Thread t holds elements 4 (t + NT j) .. +3, j < V4, of the chunk: the same ones
// whatever the row's alignment.  Every thread's largest logit is known without a
// sort; the n_out-th largest of a wave's 64 is a bound that n_out logits reach, and
// the logits that reach the largest such bound (some n_out to 3 n_out of them) are
// ranked by counting.  Where equal or unevenly spread logits leave too many, the
// n_out-th largest key of all is found bit by bit.
template <int NT, int V4>
__global__ __launch_bounds__(NT) void k_beam_part(const float* __restrict__ logits, int ld, int n_vocab,
                                                  int n_out, int vec, uint64_t* __restrict__ keys,
                                                  float* __restrict__ ms, double* __restrict__ ss) {
    constexpr int NW = NT / 64, CH = NT * V4 * 4;
    __shared__ uint64_t list[kCap];
    __shared__ double tab[32], wsum[NW];
    __shared__ uint32_t bound[NW];
    __shared__ float wm[NW];
    __shared__ int count;
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    const float* x = logits + (size_t)blockIdx.y * ld;
    const int base = blockIdx.x * CH;
    fill_exp_table(tab);
    float v[V4 * 4];
    if (vec && base + CH <= n_vocab) {
#pragma unroll
        for (int j = 0; j < V4; j++) {
            const float4 f = *reinterpret_cast<const float4*>(x + base + 4 * (t + NT * j));
            v[4 * j] = f.x;
            v[4 * j + 1] = f.y;
            v[4 * j + 2] = f.z;
            v[4 * j + 3] = f.w;
        }
    } else {
#pragma unroll
        for (int j = 0; j < V4 * 4; j++) {
            const int i = base + 4 * (t + NT * (j >> 2)) + (j & 3);
            v[j] = i < n_vocab ? x[i] : -INFINITY;
        }
    }
    float m = v[0];
#pragma unroll
    for (int j = 1; j < V4 * 4; j++) m = fmaxf(m, v[j]);
    const uint32_t mine = kth_of_wave(ordered32(m), n_out);
    m = wave_max(m);
    if (lane == 0) {
        bound[wave] = mine;
        wm[wave] = m;
    }
    if (t == 0) count = 0;
    __syncthreads();
    // -inf is no continuation's logit
    uint32_t at_least = ordered32(-__FLT_MAX__);
    m = wm[0];
#pragma unroll
    for (int w = 0; w < NW; w++) {
        at_least = max(at_least, bound[w]);
        m = fmaxf(m, wm[w]);
    }
    const float least = unordered32(at_least);
    uint32_t hits = 0;
#pragma unroll
    for (int j = 0; j < V4 * 4; j++) hits |= v[j] >= least ? 1u << j : 0;
    auto index_of = [&](int j) { return base + 4 * (t + NT * (j >> 2)) + (j & 3); };
    auto key_of = [&](int i, float y) { return ((uint64_t)ordered32(y) << 32) | (uint32_t)~i; };
    // few: read again rather than picked from registers by a variable
    for (uint32_t h = hits; h; h &= h - 1) {
        const int i = index_of(__builtin_ctz(h)), at = atomicAdd(&count, 1);
        if (at < kCap) list[at] = key_of(i, x[i]);
    }
    // sum of exponentials; a NaN or +inf logit makes it NaN, as it does the row's
    const double top = m == -INFINITY ? 0.0 : (double)m;
    double s = 0.0;
#pragma unroll
    for (int j = 0; j < V4 * 4; j++) s += exp_neg((double)v[j] - top, tab);
    s = wave_sum64(s);
    if (lane == 0) wsum[wave] = s;
    __syncthreads();
    const size_t chunk = (size_t)blockIdx.y * gridDim.x + blockIdx.x;
    if (t == 0) {
        double sum = wsum[0];
#pragma unroll
        for (int w = 1; w < NW; w++) sum += wsum[w];
        ss[chunk] = sum;
        ms[chunk] = m;
    }
    int n = count;
    if (n > kCap) {
        uint64_t c = 0;
        for (int b = 63; b >= 0; b--) {
            const uint64_t probe = c | (1ull << b);
            int r = 0;
#pragma unroll
            for (int j = 0; j < V4 * 4; j++) r += v[j] >= least && key_of(index_of(j), v[j]) >= probe;
            __syncthreads();
            if (t == 0) count = 0;
            __syncthreads();
            if (r) atomicAdd(&count, r);
            __syncthreads();
            if (count >= n_out) c = probe;
        }
        __syncthreads();
        if (t == 0) count = 0;
        __syncthreads();
        for (uint32_t h = hits; h; h &= h - 1) {
            const int i = index_of(__builtin_ctz(h));
            const uint64_t k = key_of(i, x[i]);
            if (k >= c) list[atomicAdd(&count, 1)] = k;  // keys differ: n_out of them
        }
        __syncthreads();
        n = count;
    }
    uint64_t* out = keys + chunk * n_out;
    for (int c = t; c < n; c += NT) {
        const uint64_t k = list[c];
        int rank = 0;
        for (int j = 0; j < n; j++) rank += list[j] > k;
        if (rank < n_out) out[rank] = k;
    }
    for (int c = n + t; c < n_out; c += NT) out[c] = 0;
}

// A continuation: score, and what breaks ties (beam, logit, token), both larger for
// the better; score 0: none.
struct Cand {
    uint64_t score, tie;
};
__device__ __forceinline__ bool better(const Cand& a, const Cand& b) {
    return a.score > b.score || (a.score == b.score && a.tie > b.tie);
}
__device__ __forceinline__ Cand lane_xor(const Cand& c, int x) {
    return {__shfl_xor(c.score, x, 64), __shfl_xor(c.tie, x, 64)};
}

// a and b: descending lists over the wave's lanes.  The 64 best of both, descending:
// the better of a[i] and b[63 - i] are a bitonic list of them, sorted in 6 steps.
__device__ __forceinline__ Cand merge64(Cand a, Cand b) {
    const int lane = threadIdx.x & 63;
    const Cand r = lane_xor(b, 63);
    a = better(r, a) ? r : a;
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
        const Cand o = lane_xor(a, off);
        const bool keep_max = (lane & off) == 0;
        a = (better(o, a) == keep_max) ? o : a;
    }
    return a;
}

// The k-th largest score of the wave's 64 (scores may be equal), or 0 with fewer.
__device__ __forceinline__ uint64_t kth_score(uint64_t s, int k) {
    const uint32_t hi = (uint32_t)(s >> 32), lo = (uint32_t)s, t = kth_of_wave(hi, k);
    const int above = __popcll(__ballot(hi > t));
    const bool same = hi == t;
    uint32_t v = 0;
    for (int b = 31; b >= 0; b--) {
        const uint32_t c = v | (1u << b);
        if (__popcll(__ballot(same && lo >= c)) >= k - above) v = c;
    }
    return ((uint64_t)t << 32) | v;
}

constexpr int kMergeCap = 512;    // candidates ranked at once
constexpr int kMergePicks = 512;  // lists looked into

// The chunks' lists of one sequence.  Their heads come first: a score that n_out heads
// reach bounds what can be among the n_out best, which leaves few lists and few of
// their entries (some n_out to 3 n_out candidates, ranked by counting), so that the
// rest is never read.  Many equal scores may pass the bound; then the lists are
// merged in turn, each wave a share of them.
__global__ __launch_bounds__(kMergeThreads) void k_beam_merge(
    BeamArgs a, int chunks, const uint64_t* __restrict__ keys, const float* __restrict__ ms,
    const double* __restrict__ ss) {
    constexpr int NW = kMergeThreads / 64;
    __shared__ double lse[64], cums[64];
    __shared__ int over[64];
    __shared__ Cand half[NW / 2][64];
    __shared__ Cand list[kMergeCap];
    __shared__ double tab[32];
    __shared__ uint64_t bound[NW];
    __shared__ int picks[kMergePicks];
    __shared__ uint64_t entries[kMergeThreads];
    __shared__ unsigned long long low;
    __shared__ int count, picked;
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    const size_t row0 = (size_t)blockIdx.x * a.n_beams;
    const int lists = a.n_beams * chunks;
    keys += row0 * chunks * a.n_out;
    if (t == 0) count = picked = 0;
    fill_exp_table(tab);
    if (t < a.n_beams) {
        cums[t] = (double)a.cum[row0 + t];
        over[t] = a.done && a.done[row0 + t] != 0;
    }
    // the first round's heads are in flight while the sums are joined
    const uint64_t head0 = t < lists ? keys[(size_t)t * a.n_out] : 0;
    __syncthreads();
    for (int b = wave; b < a.n_beams; b += NW) {
        const float* mr = ms + (row0 + b) * chunks;
        const double* sr = ss + (row0 + b) * chunks;
        float m0 = -INFINITY, m = -INFINITY;
        double s0 = 0.0, s = 0.0;
        if (lane < chunks) {
            m0 = mr[lane];
            s0 = sr[lane];
        }
        m = m0;
        for (int c = lane + 64; c < chunks; c += 64) m = fmaxf(m, mr[c]);
        m = wave_max(m);
        const double top = m == -INFINITY ? 0.0 : (double)m;
        s = s0 * exp_neg((double)m0 - top, tab);
        for (int c = lane + 64; c < chunks; c += 64) s += sr[c] * exp_neg((double)mr[c] - top, tab);
        s = wave_sum64(s);
        // all logits -inf: log 0, and every score -inf - -inf
        if (lane == 0) lse[b] = top + log(s);
    }
    __syncthreads();
    // list l's entry with key k (entry 0 of a finished beam's first list: its one)
    auto cand_of = [&](int l, uint64_t k, int rank) {
        const int b = l / chunks;
        Cand c = {0, 0};
        const uint64_t mine = (uint64_t)(63 - b) << 58;
        if (over[b]) {
            if (l % chunks == 0 && rank == 0 && cums[b] > -INFINITY)
                c = {ordered64(cums[b]), mine | (uint64_t)(0x3ffffff - a.eos)};
        } else if (k) {
            const uint32_t x = (uint32_t)(k >> 32);
            const double score = cums[b] + ((double)unordered32(x) - lse[b]);
            if (score > -INFINITY)
                c = {ordered64(score),
                     mine | ((uint64_t)x << 26) | (uint64_t)(0x3ffffff - ~(uint32_t)k)};
        }
        return c;
    };
    uint64_t head = 0;
    for (int l = t; l < lists; l += kMergeThreads) {
        const uint64_t s = cand_of(l, l == t ? head0 : keys[(size_t)l * a.n_out], 0).score;
        head = s > head ? s : head;
    }
    const uint64_t mine = kth_score(head, a.n_out);
    if (lane == 0) bound[wave] = mine;
    __syncthreads();
    uint64_t least = 1;
#pragma unroll
    for (int w = 0; w < NW; w++) least = bound[w] > least ? bound[w] : least;
    // The candidates that reach the bound: the lists whose head does, dealt out to the
    // waves, a lane an entry.
    int n;
    for (bool again = false;; again = true) {
        for (int l = t; l < lists; l += kMergeThreads)
            if (cand_of(l, l == t ? head0 : keys[(size_t)l * a.n_out], 0).score >= least) {
                const int at = atomicAdd(&picked, 1);
                if (at < kMergePicks) picks[at] = l;
            }
        __syncthreads();
        const int np = picked;
        for (int i = wave; i < min(np, kMergePicks); i += NW) {
            Cand c = {0, 0};
            if (lane < a.n_out) c = cand_of(picks[i], keys[(size_t)picks[i] * a.n_out + lane], lane);
            const uint64_t reach = __ballot(c.score >= least);
            int at = 0;
            if (lane == 0) at = atomicAdd(&count, __popcll(reach));
            at = __shfl(at, 0, 64) + __popcll(reach & ((1ull << lane) - 1));
            if (c.score >= least && at < kMergeCap) list[at] = c;
        }
        __syncthreads();
        n = np > kMergePicks ? kMergeCap + 1 : count;
        if (n <= kMergeCap || again) break;
        // A bound by 64 lists was too low (n_out is no small part of 64, or beams of unlike
        // scores share a wave): the n_out-th largest of 512 entries, the first few of every
        // list, by counting.  4 x 16 beams of 60000, 32 kept: 165 -> 43 us.
        const int deep = min(a.n_out, kMergeThreads / lists);
        uint64_t e = 0;
        if (deep < 1) {
            e = head;
        } else if (t < lists * deep) {
            const int l = t / deep, r = t - l * deep;
            e = cand_of(l, keys[(size_t)l * a.n_out + r], r).score;
        }
        entries[t] = e;
        __syncthreads();
        if (t == 0) {
            count = picked = 0;
            low = ~0ull;
        }
        int above = 0;
        for (int i = 0; i < kMergeThreads; i++) above += entries[i] > e;
        __syncthreads();
        if (above < a.n_out) atomicMin(&low, (unsigned long long)e);
        __syncthreads();
        least = low > least ? low : least;
    }
    const size_t o = (size_t)blockIdx.x * a.n_out;
    auto write = [&](int rank, const Cand& c) {
        const bool none = c.score == 0;
        a.token[o + rank] = none ? -1 : 0x3ffffff - (int)(c.tie & 0x3ffffff);
        a.parent[o + rank] = none ? -1 : 63 - (int)(c.tie >> 58);
        a.score[o + rank] = none ? -INFINITY : (float)unordered64(c.score);
    };
    if (n <= kMergeCap) {
        for (int i = t; i < n; i += kMergeThreads) {
            const Cand c = list[i];
            int rank = 0;
            for (int j = 0; j < n; j++) rank += better(list[j], c);
            if (rank < a.n_out) write(rank, c);
        }
        if (t >= n && t < a.n_out) write(t, Cand{0, 0});
        return;
    }
    Cand acc = {0, 0};
    for (int l = wave; l < lists; l += NW) {
        Cand c = {0, 0};
        if (lane < a.n_out) c = cand_of(l, keys[(size_t)l * a.n_out + lane], lane);
        acc = l == wave ? c : merge64(acc, c);
    }
    for (int w = NW / 2; w > 0; w >>= 1) {
        if (wave >= w && wave < 2 * w) half[wave - w][lane] = acc;
        __syncthreads();
        if (wave < w) acc = merge64(acc, half[wave][lane]);
        __syncthreads();
    }
    if (wave == 0 && lane < a.n_out) write(lane, acc);
}

constexpr int kPartThreads = 256;

// Float4s a thread: chunks of 2048 logits where few rows leave CUs idle, of 4096 (fewer
// lists to merge) from two workgroups a CU up.  8 x 8 beams of 151936: 29.0 us, with
// 2048 31.9, with 8192 (one round of waves, nothing in flight under its arithmetic) 31.4.
int beam_v4(const BeamArgs& a) {
    return (long)a.n_seq * a.n_beams * a.n_vocab >= 512L * 4096 ? 4 : 2;
}
int beam_chunks(const BeamArgs& a) {
    const int chunk = kPartThreads * 4 * beam_v4(a);
    return (a.n_vocab + chunk - 1) / chunk;
}

}  // namespace

size_t beam_scratch(const BeamArgs& a) {
    const size_t lists = (size_t)a.n_seq * a.n_beams * beam_chunks(a);
    return lists * (8 * a.n_out + 8 + 4);
}

hipError_t launch_beam_select(const BeamArgs& a, hipStream_t st) {
    const int chunks = beam_chunks(a);
    const size_t lists = (size_t)a.n_seq * a.n_beams * chunks;
    uint64_t* keys = static_cast<uint64_t*>(a.scratch);
    double* ss = reinterpret_cast<double*>(keys + lists * a.n_out);
    float* ms = reinterpret_cast<float*>(ss + lists);
    const int vec = a.ld % 4 == 0 && (reinterpret_cast<uintptr_t>(a.logits) & 15) == 0;
    const long rows = (long)a.n_seq * a.n_beams;
    // grid.y holds 65535 rows
    for (long r = 0; r < rows; r += 65535) {
        const unsigned n = (unsigned)(rows - r < 65535 ? rows - r : 65535);
        const size_t at = (size_t)r * chunks;
        auto go = [&](auto kernel) {
            kernel<<<dim3(chunks, n), kPartThreads, 0, st>>>(a.logits + (size_t)r * a.ld, a.ld,
                                                             a.n_vocab, a.n_out, vec,
                                                             keys + at * a.n_out, ms + at, ss + at);
        };
        if (beam_v4(a) == 4)
            go(k_beam_part<kPartThreads, 4>);
        else
            go(k_beam_part<kPartThreads, 2>);
    }
    k_beam_merge<<<a.n_seq, kMergeThreads, 0, st>>>(a, chunks, keys, ms, ss);
    return hipGetLastError();
}

}  // namespace axf
