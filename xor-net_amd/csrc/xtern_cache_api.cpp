// C ABI of the paged key-value cache and of the token probabilities
// (include/xtern.h): argument checks and kernel dispatch.  Every pointer,
// shape and stride is checked here; what only the device knows (lengths,
// table entries, token ids) the kernels check themselves.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>
#include <string.h>

#include <algorithm>
#include <string>

#include "../../include/xtern.h"
#include "xtern_cache.h"

// xtern_api.cpp: error message, workspace of a stream (kinds 3 and 4 are this file's),
// compute units of the current device.
int xt_internal_fail(int code, const std::string& msg);
int xt_internal_workspace(hipStream_t s, size_t bytes, void** out, int kind);
int xt_internal_cus(int* cus);

namespace {

int bad(const std::string& msg) { return xt_internal_fail(XT_ERR_INVALID, msg); }
int launched(hipError_t e, const char* what) {
    if (e == hipSuccess) return XT_OK;
    return xt_internal_fail(XT_ERR_HIP, std::string(what) + ": " + hipGetErrorString(e));
}

constexpr int64_t kMaxInt = 0x7fffffff;
constexpr int64_t kMaxLen = (int64_t)1 << 30;  // positions of a sequence
constexpr int64_t kMaxRows = (int64_t)1 << 21;  // rows of a call: a workgroup each
constexpr int kMaxGroup = 1024;                // query heads of a key-value head

int check_dtype(int dtype) {
    if (dtype != XT_F32 && dtype != XT_F16 && dtype != XT_BF16)
        return bad("unknown element type " + std::to_string(dtype));
    return XT_OK;
}

int check_align(const void* p, int size, const char* what) {
    if (reinterpret_cast<uintptr_t>(p) % (uintptr_t)size)
        return bad(std::string(what) + " is not aligned to its elements");
    return XT_OK;
}

// The cache and the table as the kernels see them.  `view` gets every field.
int check_cache(const xt_kv_cache* c, const xt_kv_table* t, xt::KvView* view) {
    if (!c || !t) return bad("cache or table is NULL");
    if (int rc = check_dtype(c->dtype)) return rc;
    if (c->head_dim < 1 || c->head_dim > 256) return bad("head_dim must be 1..256");
    if (c->kv_heads < 1 || c->kv_heads > 65535) return bad("kv_heads must be 1..65535");
    if (c->page_size < 1 || c->page_size > 65536) return bad("page_size must be 1..65536");
    if (c->num_pages < 1 || c->num_pages > kMaxInt) return bad("num_pages must be 1..2^31-1");
    if (!c->k || !c->v) return bad("NULL pointer");
    const int es = c->dtype == XT_F32 ? 4 : 2;
    if (int rc = check_align(c->k, es, "the key cache")) return rc;
    if (int rc = check_align(c->v, es, "the value cache")) return rc;
    if (int rc = check_align(c->score, 4, "the score cache")) return rc;
    // Elements of different positions must not share memory: every stride
    // covers what the smaller ones span.  (An extent of one needs no stride.)
    struct Dim {
        int64_t stride, extent;
    } d[3] = {{c->stride_page, c->num_pages}, {c->stride_slot, c->page_size}, {c->stride_head, c->kv_heads}};
    std::sort(d, d + 3, [](const Dim& x, const Dim& y) { return x.stride < y.stride; });
    int64_t span = c->head_dim;
    for (const Dim& x : d) {
        if (x.extent == 1) continue;
        if (x.stride < span) return bad("cache strides overlap");
        if (x.stride > (INT64_MAX - span) / x.extent / 4) return bad("cache strides too large");
        span += x.stride * (x.extent - 1);
    }
    if (t->seqs < 0 || t->seqs > kMaxRows) return bad("seqs must be 0..2^21");
    if (t->max_pages < 0 || t->max_pages > kMaxLen || t->max_pages * c->page_size > kMaxLen)
        return bad("max_pages * page_size must be 0..2^30");
    if (t->seqs > 0 && t->max_pages > 0 && !t->pages) return bad("NULL pointer");
    if (t->stride < t->max_pages && t->seqs > 1) return bad("table rows overlap");
    if (int rc = check_align(t->pages, 4, "the page table")) return rc;
    memset(view, 0, sizeof *view);
    view->k = c->k;
    view->v = c->v;
    view->score = c->score;
    view->sp = c->num_pages == 1 ? 0 : c->stride_page;
    view->ss = c->page_size == 1 ? 0 : c->stride_slot;
    view->sh = c->kv_heads == 1 ? 0 : c->stride_head;
    view->num_pages = (int)c->num_pages;
    view->page = c->page_size;
    view->by_page = xt::fast_div(c->page_size);
    view->hkv = c->kv_heads;
    view->D = c->head_dim;
    view->table = t->pages;
    view->ldt = t->seqs > 1 ? t->stride : 0;
    view->nseq = (int)t->seqs;
    view->max_pages = (int)t->max_pages;
    return XT_OK;
}

// R rows of `cols` f32 elements at stride ld; out: rows that are written.
int check_rows(const float* p, int64_t ld, int64_t R, int64_t cols, const char* what) {
    if (!p) return bad("NULL pointer");
    if (R > 1 && ld < cols) return bad(std::string(what) + " rows overlap");
    if (ld > INT64_MAX / 8 / std::max<int64_t>(R, 1)) return bad(std::string(what) + " stride too large");
    return check_align(p, 4, what);
}

int check_count(int64_t R) {
    if (R < 0 || R > kMaxRows) return bad("row count must be 0..2^21");
    return XT_OK;
}

int check_heads(int q_heads, int kv_heads) {
    if (q_heads < 1 || q_heads > 65535 || q_heads % kv_heads || q_heads / kv_heads > kMaxGroup)
        return bad("q_heads must be a multiple of kv_heads, 1..65535, at most 1024 times kv_heads");
    return XT_OK;
}

// Memory that no device holds (and whose size a size_t may not).
int check_fits(double bytes, const char* what) {
    if (bytes > 1e12)
        return xt_internal_fail(XT_ERR_NOMEM, std::string(what) + " would take " + std::to_string(bytes) + " bytes");
    return XT_OK;
}

// What a workspace holds for each position that the table could have (a row's
// scores, a sequence's keys) stays within this: the lengths are on the device, so a wide table
// would else take memory for positions that nobody wrote.  Calls that need more
// run in parts, one after the other in the same workspace.  4096 rows of a
// prompt with scores, 32 heads, a table for 32768 positions: 3.8 ms whole (16
// GiB), 4.2 in parts of 1 GiB, 4.1 of 2 GiB, 5.1 of 256 MiB.
constexpr int64_t kMaxScratch = (int64_t)1 << 30;
int64_t part_of(int64_t n, int64_t bytes_each) {
    const int64_t most = std::max<int64_t>(1, kMaxScratch / std::max<int64_t>(bytes_each, 1));
    const int64_t parts = (n + most - 1) / most;
    return (n + parts - 1) / parts;  // (parts of one size)
}

// The table from sequence `at` on.
void skip_sequences(xt::KvView* c, int64_t at) {
    c->table += at * c->ldt;
    c->nseq = (int)std::max<int64_t>(0, c->nseq - at);
}

// Rows [r0, r0 + n) of a call.
xt::AttnArgs rows_of(xt::AttnArgs a, int64_t r0, int64_t n) {
    a.R = n;
    a.q += r0 * a.ldq;
    a.out += r0 * a.ldo;
    if (a.lse) a.lse += r0 * a.hq;
    a.lengths += r0;
    if (a.seq) a.seq += r0;
    else skip_sequences(&a.c, r0);
    return a;
}

// At most n sequences of a call, from b0 on.
xt::EvictArgs sequences_of(xt::EvictArgs a, int64_t b0, int64_t n) {
    skip_sequences(&a.c, b0);
    a.c.nseq = (int)std::min<int64_t>(a.c.nseq, n);
    a.lengths += b0;
    a.new_lengths += b0;
    a.kept += b0 * a.c.hkv * a.budget;
    return a;
}

// The workspace and the counters of a call (either may be none).
int get_workspace(hipStream_t s, size_t bytes, size_t counters, void** ws, void** cnt) {
    *ws = *cnt = nullptr;
    if (bytes) {
        if (int rc = xt_internal_workspace(s, bytes, ws, 3)) return rc;
    }
    return counters ? xt_internal_workspace(s, counters, cnt, 4) : XT_OK;
}

}  // namespace

extern "C" {

int xt_kv_append(const xt_kv_cache* c, const xt_kv_table* t, const int32_t* seq, const int32_t* slots,
                 const int32_t* positions, const xt_rope* rope, const float* q, int64_t ldq, int q_heads,
                 float* q_out, int64_t ldqo, const float* k, int64_t ldk, const float* v, int64_t ldv,
                 int64_t R, void* stream) {
    return xt_kv_append_lengths(c, t, seq, slots, positions, rope, q, ldq, q_heads, q_out, ldqo, k, ldk, v, ldv, R,
                                nullptr, stream);
}

int xt_kv_append_lengths(const xt_kv_cache* c, const xt_kv_table* t, const int32_t* seq, const int32_t* slots,
                         const int32_t* positions, const xt_rope* rope, const float* q, int64_t ldq, int q_heads,
                         float* q_out, int64_t ldqo, const float* k, int64_t ldk, const float* v, int64_t ldv,
                         int64_t R, int32_t* lengths, void* stream) {
    xt::AppendArgs a;
    memset(&a, 0, sizeof a);
    if (int rc = check_cache(c, t, &a.c)) return rc;
    if (int rc = check_count(R)) return rc;
    if (q) {
        if (int rc = check_heads(q_heads, c->kv_heads)) return rc;
    }
    if (rope) {
        if (rope->dim < 2 || rope->dim > c->head_dim || rope->dim % 2)
            return bad("rope dim must be even, 2..head_dim");
        if (rope->rows < 0 || rope->rows > kMaxInt) return bad("rope rows must be 0..2^31-1");
        if (!rope->cos || !rope->sin) return bad("NULL pointer");
        if (int rc = check_align(rope->cos, 4, "cos")) return rc;
        if (int rc = check_align(rope->sin, 4, "sin")) return rc;
    }
    if (R == 0) return XT_OK;
    if (!slots) return bad("NULL pointer");
    const int64_t D = c->head_dim;
    if (int rc = check_rows(k, ldk, R, c->kv_heads * D, "k")) return rc;
    if (int rc = check_rows(v, ldv, R, c->kv_heads * D, "v")) return rc;
    if (q) {
        if (int rc = check_rows(q, ldq, R, q_heads * D, "q")) return rc;
        if (int rc = check_rows(q_out, ldqo, R, q_heads * D, "q_out")) return rc;
        if (q == q_out && ldq != ldqo && R > 1) return bad("q_out overlaps q at another stride");
    }
    if (int rc = check_align(lengths, 4, "lengths")) return rc;
    if (lengths && (lengths == slots || lengths == seq || lengths == positions))
        return bad("lengths must not be slots, seq or positions");
    a.lengths = lengths;
    a.seq = seq;
    a.slots = slots;
    a.pos = positions ? positions : slots;
    if (rope) {
        a.cos = rope->cos;
        a.sin = rope->sin;
        a.rope_rows = rope->rows;
        a.rot = rope->dim;
    }
    a.q = q;
    a.qo = q_out;
    a.ldq = ldq;
    a.ldqo = ldqo;
    a.hq = q ? q_heads : 0;
    a.k = k;
    a.v = v;
    a.ldk = ldk;
    a.ldv = ldv;
    a.R = R;
    return launched(xt::launch_kv_append(c->dtype, a, static_cast<hipStream_t>(stream)), "cache append launch");
}

int xt_paged_attention(const xt_kv_cache* c, const xt_kv_table* t, const int32_t* seq, const int32_t* lengths,
                       const float* q, int64_t ldq, int q_heads, float scale, int64_t R, float* out, int64_t ldo,
                       float* lse, int accumulate, void* stream) {
    xt::AttnArgs a;
    memset(&a, 0, sizeof a);
    if (int rc = check_cache(c, t, &a.c)) return rc;
    if (int rc = check_count(R)) return rc;
    if (int rc = check_heads(q_heads, c->kv_heads)) return rc;
    // (the kernels work with scale in base 2)
    if (!isfinite((float)((double)scale * 1.4426950408889634))) return bad("scale must be finite, at most 2.3e38");
    if (accumulate && !c->score) return bad("accumulate needs a cache with scores");
    if (R == 0) return XT_OK;
    if (!lengths) return bad("NULL pointer");
    const int64_t cols = (int64_t)q_heads * c->head_dim;
    if (int rc = check_rows(q, ldq, R, cols, "q")) return rc;
    if (int rc = check_rows(out, ldo, R, cols, "out")) return rc;
    if (int rc = check_align(lse, 4, "lse")) return rc;
    // (in place is fine: the workgroups that read a row's head have read it
    // before the one that writes it does)
    if (q == out && ldq != ldo && R > 1) return bad("out overlaps q at another stride");
    a.seq = seq;
    a.lengths = lengths;
    a.q = q;
    a.ldq = ldq;
    a.hq = q_heads;
    a.scale = scale;
    a.R = a.call_rows = R;
    a.out = out;
    a.ldo = ldo;
    a.lse = lse;
    a.accumulate = accumulate ? 1 : 0;
    int64_t part = R;  // rows at a time
    if (a.accumulate) {
        const int64_t row = 4 * (int64_t)q_heads * t->max_pages * c->page_size;
        part = part_of(R, row);
        if (int rc = check_fits((double)part * (double)row, "the workspace")) return rc;
    }
    int cus = 0;
    if (int rc = xt_internal_cus(&cus)) return rc;
    hipStream_t st = static_cast<hipStream_t>(stream);
    void *ws, *counters;
    size_t nc, nc_last;
    const xt::AttnArgs last = rows_of(a, (R - 1) / part * part, R - (R - 1) / part * part);
    const size_t bytes_last = xt::attention_workspace(last, cus, &nc_last);
    const size_t bytes = std::max(bytes_last, xt::attention_workspace(rows_of(a, 0, part), cus, &nc));
    if (int rc = get_workspace(st, bytes, std::max(nc, nc_last), &ws, &counters)) return rc;
    for (int64_t r0 = 0; r0 < R; r0 += part) {
        const xt::AttnArgs b = rows_of(a, r0, std::min(part, R - r0));
        if (int rc = launched(xt::launch_paged_attention(c->dtype, b, cus, ws, counters, st), "paged attention launch"))
            return rc;
    }
    return XT_OK;
}

int xt_kv_evict(const xt_kv_cache* c, const xt_kv_table* t, const int32_t* lengths, int64_t budget, int64_t sink,
                int64_t recent, int32_t* new_lengths, int32_t* kept, void* stream) {
    xt::EvictArgs a;
    memset(&a, 0, sizeof a);
    if (int rc = check_cache(c, t, &a.c)) return rc;
    if (!c->score) return bad("eviction needs a cache with scores");
    if (budget < 1 || budget > kMaxInt) return bad("budget must be 1..2^31-1");
    if (sink < 0 || recent < 0 || sink > budget || recent > budget - sink)
        return bad("sink and recent must be >= 0, their sum at most budget");
    if (t->seqs == 0) return XT_OK;
    if (!lengths || !new_lengths || !kept) return bad("NULL pointer");
    if (new_lengths == lengths) return bad("new_lengths must not be lengths");
    a.lengths = lengths;
    a.new_lengths = new_lengths;
    a.kept = kept;
    a.budget = (int)budget;
    a.sink = (int)sink;
    a.recent = (int)recent;
    const int64_t keys = (int64_t)xt::evict_key_bytes(a), part = part_of(t->seqs, keys);  // sequences at a time
    if (int rc = check_fits(4.0 * (double)t->seqs * (double)t->max_pages, "the page table")) return rc;
    if (int rc = check_fits((double)keys, "the workspace")) return rc;
    int cus = 0;
    if (int rc = xt_internal_cus(&cus)) return rc;
    hipStream_t st = static_cast<hipStream_t>(stream);
    void *ws, *counters;
    const size_t bytes_last = xt::evict_workspace(c->dtype, sequences_of(a, (t->seqs - 1) / part * part, part), cus);
    const size_t bytes = std::max(bytes_last, xt::evict_workspace(c->dtype, sequences_of(a, 0, part), cus));
    if (int rc = get_workspace(st, bytes, 0, &ws, &counters)) return rc;
    for (int64_t b0 = 0; b0 < t->seqs; b0 += part)
        if (int rc = launched(xt::launch_kv_evict(c->dtype, sequences_of(a, b0, part), cus, ws, st),
                              "cache eviction launch"))
            return rc;
    return XT_OK;
}

int xt_token_logprobs(int dtype, const void* logits, int64_t ld, int64_t M, int64_t V, const int32_t* tokens,
                      int64_t T, float* logprobs, float* entropy, int top, int32_t* top_ids, float* top_logprobs,
                      void* stream) {
    if (int rc = check_dtype(dtype)) return rc;
    if (int rc = check_count(M)) return rc;
    if (V < 1 || V > (1 << 30)) return bad("vocabulary must be 1..2^30");
    if (T < 0 || T > (1 << 20)) return bad("tokens per row must be 0..2^20");
    if (top < 0 || top > 64 || top > V) return bad("top must be 0..64, at most the vocabulary");
    if (M == 0) return XT_OK;
    if (!logits || !entropy || (T > 0 && (!tokens || !logprobs)) || (top > 0 && (!top_ids || !top_logprobs)))
        return bad("NULL pointer");
    if (M > 1 && ld < V) return bad("logits rows overlap");
    if (M > 1 && ld > INT64_MAX / 8 / M) return bad("logits stride too large");
    if (int rc = check_align(logits, dtype == XT_F32 ? 4 : 2, "logits")) return rc;
    xt::ProbsArgs a;
    memset(&a, 0, sizeof a);
    a.x = logits;
    a.ld = M > 1 ? ld : 0;
    a.M = M;
    a.V = (int)V;
    a.tokens = tokens;
    a.T = (int)T;
    a.lp = logprobs;
    a.entropy = entropy;
    a.top = top;
    a.ids = top_ids;
    a.top_lp = top_logprobs;
    int cus = 0;
    if (int rc = xt_internal_cus(&cus)) return rc;
    hipStream_t st = static_cast<hipStream_t>(stream);
    void *ws, *counters;
    size_t nc;
    const size_t bytes = xt::token_logprobs_workspace(a, cus, &nc);
    if (int rc = get_workspace(st, bytes, nc, &ws, &counters)) return rc;
    return launched(xt::launch_token_logprobs(dtype, a, cus, ws, counters, st),
                    "token probabilities launch");
}

}  // extern "C"
