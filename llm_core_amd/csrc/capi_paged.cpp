// capi_paged.cpp — C-ABI entry points of the cache in pages and of beam search
// (declared in include/axf_hip.h; kernels in kernels/paged.hip, kernels/beam.hip).
#include "capi_check.hpp"

#include <initializer_list>
#include <string>

using namespace axf;

namespace {

// What is wrong with a page pool, or nullptr.
const char* pages_fault(const axf_kv_pages* kv) {
    if (!kv || !kv->k || !kv->v) return "null page pool";
    if (kv->type != AXF_TYPE_F32 && kv->type != AXF_TYPE_F16) return "pages must be F32 or F16";
    if (kv->head_dim != 64 && kv->head_dim != 128 && kv->head_dim != 256)
        return "head_dim must be 64, 128 or 256";
    if (kv->n_layers <= 0 || kv->n_layers > 16384 || kv->n_pages <= 0 || kv->n_kv_heads <= 0 ||
        kv->n_kv_heads > 256)
        return "bad pool shape";
    if (kv->page_rows <= 0 || kv->page_rows > 1024 || (kv->page_rows & (kv->page_rows - 1)))
        return "page_rows must be a power of two up to 1024";
    if ((long)kv->n_pages * kv->page_rows > 0x7fffffffL) return "more than 2^31 rows a layer";
    if (!aligned(kv->k, 16) || !aligned(kv->v, 16)) return "pages must be 16-byte aligned";
    return nullptr;
}

int page_shift(const axf_kv_pages* kv) { return __builtin_ctz((unsigned)kv->page_rows); }

size_t layer_bytes(const axf_kv_pages* kv) {
    return (size_t)kv->n_pages * kv->page_rows * kv->n_kv_heads * kv->head_dim *
           (kv->type == AXF_TYPE_F32 ? 4 : 2);
}

// An argument's array, for fault messages by name.  None (a null pointer) has no bytes.
struct Array {
    const char* name;
    const void* p;
    size_t bytes;
};

// What is wrong where a call writes arrays that it also reads (other workgroups may do so
// later) or writes as something else: empty if nothing.
std::string overlap_fault(std::initializer_list<Array> writes, std::initializer_list<Array> reads) {
    auto common = [](const Array& a, const Array& b) {
        const uintptr_t x = reinterpret_cast<uintptr_t>(a.p), y = reinterpret_cast<uintptr_t>(b.p);
        return a.p && b.p && x < y + b.bytes && y < x + a.bytes;
    };
    for (const Array* w = writes.begin(); w != writes.end(); w++) {
        for (const Array* o = w + 1; o != writes.end(); o++)
            if (common(*w, *o)) return std::string(w->name) + " must not overlap " + o->name;
        for (const Array& r : reads)
            if (common(*w, r)) return std::string(w->name) + " must not overlap " + r.name;
    }
    return {};
}
#define AXF_REQUIRE_APART(...)                                            \
    do {                                                                  \
        const std::string fault_ = overlap_fault(__VA_ARGS__);            \
        AXF_REQUIRE(fault_.empty(), fault_);                              \
    } while (0)

// Positions are 32-bit.
bool table_ok(const axf_kv_pages* kv, int table_ld) {
    return table_ld > 0 && ((long)table_ld << page_shift(kv)) <= (1L << 30);
}

}  // namespace

extern "C" {

int axf_tree_masks(uint64_t* mask, int32_t* depth, const int32_t* parent, int n) {
    AXF_REQUIRE(mask && parent && n > 0 && n <= 64, "bad arguments (1 to 64 nodes)");
    uint64_t m[64];  // written once parent is read: it may be the same memory
    int32_t d[64];
    for (int i = 0; i < n; i++) {
        const int32_t p = parent[i];
        AXF_REQUIRE(p >= -1 && p < i, "a node's parent must come before it");
        m[i] = (1ull << i) | (p >= 0 ? m[p] : 0);
        d[i] = p >= 0 ? d[p] + 1 : 0;
    }
    for (int i = 0; i < n; i++) {
        mask[i] = m[i];
        if (depth) depth[i] = d[i];
    }
    return AXF_OK;
}

int axf_hip_kv_fork(axf_ctx* ctx, const axf_kv_pages* kv, int32_t* table_out, int32_t* refs_out,
                    int32_t* info, const int32_t* table, const int32_t* refs, int n_in,
                    const int32_t* parent, const int32_t* len, int n_out, int table_ld,
                    int extra) {
    AXF_CHECK_CTX(ctx);
    if (const char* f = pages_fault(kv)) AXF_REQUIRE(false, f);
    AXF_REQUIRE(n_in >= 0 && n_out >= 0 && n_in <= 65536 && n_out <= 65536,
                "up to 65536 sequences");
    AXF_REQUIRE(table_ok(kv, table_ld), "bad table_ld");
    // the kernel steps over its pages, 4096 at a time, in 32 bits
    AXF_REQUIRE(kv->n_pages <= (1 << 30), "a pool of more than 2^30 pages");
    // the kernel counts pages to take in 32 bits
    AXF_REQUIRE((long)n_out * table_ld < (1L << 31), "table_out of 2^31 entries or more");
    AXF_REQUIRE(extra >= 0 && extra <= (1 << 30), "bad extra");
    AXF_REQUIRE(refs && refs_out && info && (n_in == 0 || table) &&
                    (n_out == 0 || (table_out && parent && len)),
                "null pointer");
    AXF_REQUIRE(aligned(table, 4) && aligned(table_out, 4) && aligned(refs, 4) &&
                    aligned(refs_out, 4) && aligned(info, 4) && aligned(parent, 4) &&
                    aligned(len, 4),
                "misaligned pointer");
    const size_t entry = (size_t)table_ld * 4, seqs = (size_t)n_out * 4;
    const size_t pool = extra > 0 ? kv->n_layers * layer_bytes(kv) : 0;  // 0: not touched
    AXF_REQUIRE_APART({{"table_out", table_out, n_out * entry},
                       {"refs_out", refs_out, (size_t)kv->n_pages * 4},
                       {"info", info, 12},
                       {"k", pool ? kv->k : nullptr, pool},
                       {"v", pool ? kv->v : nullptr, pool}},
                      {{"table", table, n_in * entry},
                       {"refs", refs == refs_out ? nullptr : refs, (size_t)kv->n_pages * 4},
                       {"parent", parent, seqs},
                       {"len", len, seqs}});
    DeviceScope device(ctx);
    void* scratch = nullptr;
    int rc = ctx_scratch(ctx, kv_fork_scratch(kv->n_pages, n_out), &scratch);
    if (rc) return rc;
    KvForkArgs a{};
    a.table_out = table_out;
    a.refs_out = refs_out;
    a.info = info;
    a.table = table;
    a.refs = refs;
    a.parent = parent;
    a.len = len;
    a.n_in = n_in;
    a.n_out = n_out;
    a.table_ld = table_ld;
    a.extra = extra;
    a.n_pages = kv->n_pages;
    a.page_shift = page_shift(kv);
    a.scratch = static_cast<int*>(scratch);
    AXF_HIP(launch_kv_fork(a, *kv, ctx->stream));
    return AXF_OK;
}

int axf_hip_kv_store(axf_ctx* ctx, const axf_kv_pages* kv, int layer, const int32_t* table,
                     int table_ld, const int32_t* len, const int32_t* n_tok, int n_seq,
                     int max_tok, const float* k, int k_ld, const float* bk, const float* v,
                     int v_ld, const float* bv, const int32_t* pos, const float* cos_t,
                     const float* sin_t, int n_pos) {
    AXF_CHECK_CTX(ctx);
    if (const char* f = pages_fault(kv)) AXF_REQUIRE(false, f);
    AXF_REQUIRE(layer >= 0 && layer < kv->n_layers, "layer out of range");
    AXF_REQUIRE(table_ok(kv, table_ld), "bad table_ld");
    AXF_REQUIRE(n_seq >= 0 && max_tok >= 0 && (long)n_seq * max_tok <= (1L << 24),
                "bad token counts");
    if (n_seq == 0 || max_tok == 0) return AXF_OK;
    AXF_REQUIRE(table && len && k && v, "null pointer");
    AXF_REQUIRE(!pos || (cos_t && sin_t && n_pos > 0), "pos needs the RoPE tables");
    const int row = kv->n_kv_heads * kv->head_dim;
    AXF_REQUIRE(k_ld >= row && v_ld >= row, "k_ld or v_ld below one row");
    AXF_REQUIRE(aligned(table, 4) && aligned(len, 4) && aligned(n_tok, 4) && aligned(k, 4) &&
                    aligned(v, 4) && aligned(bk, 4) && aligned(bv, 4) && aligned(pos, 4) &&
                    aligned(cos_t, 4) && aligned(sin_t, 4),
                "misaligned pointer");
    const size_t bytes = layer_bytes(kv), rows = (size_t)n_seq * max_tok, seqs = (size_t)n_seq * 4;
    const size_t turns = (size_t)n_pos * (kv->head_dim / 2) * 4;
    char* const k_at = static_cast<char*>(kv->k) + layer * bytes;
    char* const v_at = static_cast<char*>(kv->v) + layer * bytes;
    AXF_REQUIRE_APART({{"the pages' k", k_at, bytes}, {"the pages' v", v_at, bytes}},
                      {{"table", table, seqs * table_ld},
                       {"len", len, seqs},
                       {"n_tok", n_tok, seqs},
                       {"k", k, ((rows - 1) * k_ld + row) * 4},
                       {"bk", bk, (size_t)row * 4},
                       {"v", v, ((rows - 1) * v_ld + row) * 4},
                       {"bv", bv, (size_t)row * 4},
                       {"pos", pos, rows * 4},
                       {"cos_t", pos ? cos_t : nullptr, turns},
                       {"sin_t", pos ? sin_t : nullptr, turns}});
    DeviceScope device(ctx);
    KvStoreArgs a{};
    a.k = k_at;
    a.v = v_at;
    a.table = table;
    a.table_ld = table_ld;
    a.len = len;
    a.n_tok = n_tok;
    a.pos = pos;
    a.xk = k;
    a.xv = v;
    a.bk = bk;
    a.bv = bv;
    a.cos_t = cos_t;
    a.sin_t = sin_t;
    a.k_ld = k_ld;
    a.v_ld = v_ld;
    a.n_pos = n_pos;
    a.n_seq = n_seq;
    a.max_tok = max_tok;
    a.n_kv_heads = kv->n_kv_heads;
    a.n_pages = kv->n_pages;
    a.page_shift = page_shift(kv);
    AXF_HIP(launch_kv_store(a, kv->type, kv->head_dim, ctx->stream));
    return AXF_OK;
}

int axf_hip_attn_paged(axf_ctx* ctx, float* out, void* outq8, const float* q, int q_ld,
                       const float* bq, const axf_kv_pages* kv, int layer, const int32_t* table,
                       int table_ld, const int32_t* len, const int32_t* n_tok,
                       const uint64_t* mask, const int32_t* pos, const float* cos_t,
                       const float* sin_t, int n_pos, int n_seq, int max_tok, int max_len,
                       int n_heads) {
    AXF_CHECK_CTX(ctx);
    if (const char* f = pages_fault(kv)) AXF_REQUIRE(false, f);
    AXF_REQUIRE(layer >= 0 && layer < kv->n_layers, "layer out of range");
    AXF_REQUIRE(table_ok(kv, table_ld), "bad table_ld");
    AXF_REQUIRE(n_heads > 0 && n_heads <= 1024 && n_heads % kv->n_kv_heads == 0,
                "n_heads must be a multiple of n_kv_heads up to 1024");
    AXF_REQUIRE(max_tok >= 0 && max_tok <= 64, "at most 64 tokens a sequence");
    AXF_REQUIRE(n_seq >= 0 && n_seq <= 65536 && max_len >= 0, "bad sizes");
    AXF_REQUIRE((long)n_seq * max_tok * n_heads <= (1L << 26), "too many query rows");
    if (n_seq == 0 || max_tok == 0) return AXF_OK;
    AXF_REQUIRE(out && q && table && len, "null pointer");
    AXF_REQUIRE(!pos || (cos_t && sin_t && n_pos > 0), "pos needs the RoPE tables");
    AXF_REQUIRE(q_ld >= n_heads * kv->head_dim, "q_ld below one row");
    AXF_REQUIRE(aligned(out, 4) && aligned(outq8, 4) && aligned(q, 4) && aligned(bq, 4) &&
                    aligned(table, 4) && aligned(len, 4) && aligned(n_tok, 4) &&
                    aligned(mask, 8) && aligned(pos, 4) && aligned(cos_t, 4) && aligned(sin_t, 4),
                "misaligned pointer");
    const size_t rows = (size_t)n_seq * max_tok, row = (size_t)n_heads * kv->head_dim;
    const size_t bytes = layer_bytes(kv), seqs = (size_t)n_seq * 4;
    const size_t turns = (size_t)n_pos * (kv->head_dim / 2) * 4;
    const char* const k_at = static_cast<const char*>(kv->k) + layer * bytes;
    const char* const v_at = static_cast<const char*>(kv->v) + layer * bytes;
    AXF_REQUIRE_APART({{"out", out, rows * row * 4}, {"outq8", outq8, rows * (row / 32) * Q8_0_BYTES}},
                      {{"q", q, ((rows - 1) * q_ld + row) * 4},
                       {"bq", bq, row * 4},
                       {"the pages' k", k_at, bytes},
                       {"the pages' v", v_at, bytes},
                       {"table", table, seqs * table_ld},
                       {"len", len, seqs},
                       {"n_tok", n_tok, seqs},
                       {"mask", mask, rows * 8},
                       {"pos", pos, rows * 4},
                       {"cos_t", pos ? cos_t : nullptr, turns},
                       {"sin_t", pos ? sin_t : nullptr, turns}});
    DeviceScope device(ctx);
    PagedArgs a{};
    a.q = q;
    a.q_ld = q_ld;
    a.bq = bq;
    a.k = k_at;
    a.v = v_at;
    a.table = table;
    a.table_ld = table_ld;
    a.len = len;
    a.n_tok = n_tok;
    a.mask = mask;
    a.pos = pos;
    a.cos_t = cos_t;
    a.sin_t = sin_t;
    a.n_pos = n_pos;
    a.n_seq = n_seq;
    a.max_tok = max_tok;
    a.n_heads = n_heads;
    a.n_kv_heads = kv->n_kv_heads;
    a.group = n_heads / kv->n_kv_heads;
    a.n_pages = kv->n_pages;
    a.page_shift = page_shift(kv);
    a.out = out;
    a.outq8 = static_cast<uint8_t*>(outq8);
    attn_paged_plan(a, kv->type, kv->head_dim, max_len);
    void* scratch = nullptr;
    int rc = ctx_scratch(ctx, attn_paged_scratch(a, kv->type, kv->head_dim), &scratch);
    if (rc) return rc;
    AXF_HIP(launch_attn_paged(a, kv->type, kv->head_dim, scratch, ctx->stream));
    return AXF_OK;
}

int axf_hip_kv_compact(axf_ctx* ctx, const axf_kv_pages* kv, int32_t* len_out,
                       const int32_t* table, int table_ld, const int32_t* len,
                       const int32_t* path, const int32_t* n_path, int n_seq, int max_path) {
    AXF_CHECK_CTX(ctx);
    if (const char* f = pages_fault(kv)) AXF_REQUIRE(false, f);
    AXF_REQUIRE(table_ok(kv, table_ld), "bad table_ld");
    AXF_REQUIRE(max_path >= 0 && max_path <= 64, "at most 64 rows a path");
    AXF_REQUIRE(n_seq >= 0 && n_seq <= 65535, "bad n_seq");
    if (n_seq == 0) return AXF_OK;
    AXF_REQUIRE(len_out && table && len && n_path && (path || max_path == 0), "null pointer");
    AXF_REQUIRE(aligned(len_out, 4) && aligned(table, 4) && aligned(len, 4) && aligned(path, 4) &&
                    aligned(n_path, 4),
                "misaligned pointer");
    const size_t seqs = (size_t)n_seq * 4;
    const size_t pool = max_path > 0 ? kv->n_layers * layer_bytes(kv) : 0;  // 0: not touched
    AXF_REQUIRE_APART({{"len_out", len_out, seqs},
                       {"k", pool ? kv->k : nullptr, pool},
                       {"v", pool ? kv->v : nullptr, pool}},
                      {{"table", table, seqs * table_ld},
                       {"len", len == len_out ? nullptr : len, seqs},
                       {"path", path, seqs * max_path},
                       {"n_path", n_path, seqs}});
    DeviceScope device(ctx);
    AXF_HIP(launch_kv_compact(*kv, len_out, table, table_ld, len, path, n_path, n_seq, max_path,
                              ctx->stream));
    return AXF_OK;
}

int axf_hip_beam_select(axf_ctx* ctx, int32_t* token, int32_t* parent, float* score,
                        const float* logits, int ld, const float* cum, const int32_t* done,
                        int eos_id, int n_seq, int n_beams, int n_vocab, int n_out) {
    AXF_CHECK_CTX(ctx);
    AXF_REQUIRE(n_beams > 0 && n_beams <= 64, "1 to 64 beams");
    AXF_REQUIRE(n_out > 0 && n_out <= 64, "1 to 64 continuations");
    AXF_REQUIRE(n_vocab > 0 && n_vocab <= (1 << 26), "n_vocab out of range");
    AXF_REQUIRE(n_seq >= 0 && n_seq <= 16384, "bad n_seq");
    AXF_REQUIRE(ld >= n_vocab, "ld below one row");
    if (n_seq == 0) return AXF_OK;
    AXF_REQUIRE(token && parent && score && logits && cum, "null pointer");
    AXF_REQUIRE(!done || (eos_id >= 0 && eos_id < n_vocab), "eos_id out of range");
    AXF_REQUIRE(aligned(token, 4) && aligned(parent, 4) && aligned(score, 4) &&
                    aligned(logits, 4) && aligned(cum, 4) && aligned(done, 4),
                "misaligned pointer");
    const size_t rows = (size_t)n_seq * n_beams, kept = (size_t)n_seq * n_out * 4;
    AXF_REQUIRE_APART({{"token", token, kept}, {"parent", parent, kept}, {"score", score, kept}},
                      {{"logits", logits, ((rows - 1) * ld + n_vocab) * 4},
                       {"cum", score == cum && n_out == n_beams ? nullptr : cum, rows * 4},
                       {"done", done, rows * 4}});
    DeviceScope device(ctx);
    BeamArgs a{};
    a.token = token;
    a.parent = parent;
    a.score = score;
    a.logits = logits;
    a.cum = cum;
    a.done = done;
    a.ld = ld;
    a.eos = eos_id;
    a.n_seq = n_seq;
    a.n_beams = n_beams;
    a.n_vocab = n_vocab;
    a.n_out = n_out;
    void* scratch = nullptr;
    int rc = ctx_scratch(ctx, beam_scratch(a), &scratch);
    if (rc) return rc;
    a.scratch = scratch;
    AXF_HIP(launch_beam_select(a, ctx->stream));
    return AXF_OK;
}

}  // extern "C"
