// C ABI of the paged key-value cache, of the token probabilities and of the
// verification of drafted tokens (include/xtern.h): argument checks and kernel dispatch.  Every pointer,
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

// The cache (whose scales go with an XT_I8 one) and the table as the kernels see
// them.  `view` gets every field.
int check_cache(const xt_kv_cache* c, const xt_kv_scales* scales, const xt_kv_table* t, xt::KvView* view) {
    if (!c || !t) return bad("cache or table is NULL");
    const bool codes = c->dtype == XT_I8;
    if (codes) {
        if (!scales) return bad("a cache of 8-bit codes needs its scales");
        if (!scales->k || !scales->v) return bad("NULL pointer");
        if (c->score) return bad("a cache of 8-bit codes keeps no score");
        if (int rc = check_align(scales->k, 4, "the key scales")) return rc;
        if (int rc = check_align(scales->v, 4, "the value scales")) return rc;
    } else {
        if (int rc = check_dtype(c->dtype)) return rc;
        if (scales) return bad("scales belong to a cache of 8-bit codes");
    }
    if (c->head_dim < 1 || c->head_dim > 256) return bad("head_dim must be 1..256");
    if (c->kv_heads < 1 || c->kv_heads > 65535) return bad("kv_heads must be 1..65535");
    if (c->page_size < 1 || c->page_size > 65536) return bad("page_size must be 1..65536");
    if (c->num_pages < 1 || c->num_pages > kMaxInt) return bad("num_pages must be 1..2^31-1");
    if (!c->k || !c->v) return bad("NULL pointer");
    const int es = codes ? 1 : (c->dtype == XT_F32 ? 4 : 2);
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

template <typename Args>
void set_scales(const xt_kv_scales* scales, Args* a) {
    a->ks = scales ? scales->k : nullptr;
    a->vs = scales ? scales->v : nullptr;
}

// R rows of `cols` elements (f32, or of `size` bytes) at stride ld.
int check_rows(const void* p, int64_t ld, int64_t R, int64_t cols, const char* what, int size = 4) {
    if (!p) return bad("NULL pointer");
    if (R > 1 && ld < cols) return bad(std::string(what) + " rows overlap");
    if (ld > INT64_MAX / 8 / std::max<int64_t>(R, 1)) return bad(std::string(what) + " stride too large");
    return check_align(p, size, what);
}

// [S][rows] rows of V logits of `size` bytes; they may overlap (one row shown to
// several sequences).
int check_logits(const void* p, int64_t ld_seq, int64_t ld_row, int64_t S, int64_t rows, int64_t V, const char* what,
                 int size) {
    const int64_t most = INT64_MAX / 16;
    if ((S > 1 && (ld_seq < 0 || ld_seq > most / S)) || (rows > 1 && (ld_row < 0 || ld_row > most / rows)))
        return bad(std::string(what) + " strides must not be negative or too large");
    return check_align(p, size, what);
}

// Whether [out, out + bytes) shares memory with a row of those.
bool meets_logits(uintptr_t out, uint64_t bytes, const void* p, int64_t ld_seq, int64_t ld_row, int64_t S, int64_t rows,
                  int64_t V, int size) {
    const uint64_t row = (uint64_t)V * size, by_row = rows > 1 ? (uint64_t)ld_row * size : 0;
    const uint64_t by_seq = S > 1 ? (uint64_t)ld_seq * size : 0, last = (uint64_t)S - 1;
    const uintptr_t first = reinterpret_cast<uintptr_t>(p);
    if (out + bytes <= first || out >= first + last * by_seq + (uint64_t)(rows - 1) * by_row + row) return false;
    for (int64_t j = 0; j < rows; ++j) {
        const uintptr_t at = first + (uint64_t)j * by_row;
        if (out + bytes <= at) break;  // (all of them begin behind it)
        // the last sequence whose row begins before out's end: the others' end earlier
        const uint64_t i = by_seq ? std::min(last, (out + bytes - 1 - at) / by_seq) : 0;
        if (at + i * by_seq + row > out) return true;
    }
    return false;
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
    if (a.tokens > 1) a.row0 = (int)r0;  // (groups: seq and table as they are)
    else if (a.seq) a.seq += r0;
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

// The arguments of an append, of R > 0 rows where it returns XT_OK.
int append_args(const xt_kv_cache* c, const xt_kv_scales* scales, const xt_kv_table* t, const int32_t* seq,
                const int32_t* slots, const int32_t* positions, const xt_rope* rope, const xt_head_norm* norm,
                const float* q, int64_t ldq, int q_heads, float* q_out, int64_t ldqo, const float* k, int64_t ldk,
                const float* v, int64_t ldv, int64_t R, int32_t* lengths, xt::AppendArgs* args) {
    xt::AppendArgs& a = *args;
    memset(&a, 0, sizeof a);
    if (int rc = check_cache(c, scales, t, &a.c)) return rc;
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
    if (norm) {
        if (!norm->k || (q && !norm->q)) return bad("NULL pointer");
        if (!(norm->eps >= 0.0) || !isfinite(norm->eps)) return bad("norm eps must be finite, >= 0");
        if (int rc = check_align(norm->q, 4, "the query norm")) return rc;
        if (int rc = check_align(norm->k, 4, "the key norm")) return rc;
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
    set_scales(scales, &a);
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
    if (norm) {
        a.q_norm = norm->q;
        a.k_norm = norm->k;
        a.eps = norm->eps;
    }
    return XT_OK;
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
    if (int rc = append_args(c, nullptr, t, seq, slots, positions, rope, nullptr, q, ldq, q_heads, q_out, ldqo, k, ldk,
                             v, ldv, R, lengths, &a))
        return rc;
    if (R == 0) return XT_OK;
    return launched(xt::launch_kv_append(c->dtype, a, static_cast<hipStream_t>(stream)), "cache append launch");
}

int xt_kv_store(const xt_kv_cache* c, const xt_kv_scales* scales, const xt_kv_table* t, const int32_t* seq,
                const int32_t* slots, const int32_t* positions, const xt_rope* rope, const xt_head_norm* norm,
                const float* q, int64_t ldq, int q_heads, float* q_out, int64_t ldqo, const float* k, int64_t ldk,
                const float* v, int64_t ldv, int64_t R, int32_t* lengths, void* stream) {
    xt::AppendArgs a;
    if (int rc = append_args(c, scales, t, seq, slots, positions, rope, norm, q, ldq, q_heads, q_out, ldqo, k, ldk, v,
                             ldv, R, lengths, &a))
        return rc;
    if (R == 0) return XT_OK;
    int cus = 0;
    if (int rc = xt_internal_cus(&cus)) return rc;
    return launched(xt::launch_kv_store(c->dtype, a, cus, static_cast<hipStream_t>(stream)), "cache store launch");
}

int xt_kv_read(const xt_kv_cache* c, const xt_kv_scales* scales, const xt_kv_table* t, const int32_t* seq,
               const int32_t* slots, int64_t R, int out, void* k, int64_t ldk, void* v, int64_t ldv, void* stream) {
    xt::ReadArgs a;
    memset(&a, 0, sizeof a);
    if (int rc = check_cache(c, scales, t, &a.c)) return rc;
    if (int rc = check_dtype(out)) return rc;
    if (int rc = check_count(R)) return rc;
    if (R == 0) return XT_OK;
    if (!slots) return bad("NULL pointer");
    const int64_t cols = (int64_t)c->kv_heads * c->head_dim;
    const int es = out == XT_F32 ? 4 : 2;
    if (int rc = check_rows(k, ldk, R, cols, "k", es)) return rc;
    if (int rc = check_rows(v, ldv, R, cols, "v", es)) return rc;
    set_scales(scales, &a);
    a.seq = seq;
    a.slots = slots;
    a.k = k;
    a.v = v;
    a.ldk = ldk;
    a.ldv = ldv;
    a.R = R;
    int cus = 0;
    if (int rc = xt_internal_cus(&cus)) return rc;
    return launched(xt::launch_kv_read(c->dtype, out, a, cus, static_cast<hipStream_t>(stream)), "cache read launch");
}

int xt_paged_attention(const xt_kv_cache* c, const xt_kv_table* t, const int32_t* seq, const int32_t* lengths,
                       const float* q, int64_t ldq, int q_heads, float scale, int64_t R, float* out, int64_t ldo,
                       float* lse, int accumulate, void* stream) {
    return xt_paged_attention_window(c, nullptr, t, seq, lengths, 1, 0, 0, q, ldq, q_heads, scale, R, out, ldo, lse,
                                     accumulate, stream);
}

int xt_paged_attention_window(const xt_kv_cache* c, const xt_kv_scales* scales, const xt_kv_table* t,
                              const int32_t* seq, const int32_t* lengths, int64_t tokens, int64_t window,
                              int64_t sink, const float* q, int64_t ldq, int q_heads, float scale, int64_t R,
                              float* out, int64_t ldo, float* lse, int accumulate, void* stream) {
    xt::AttnArgs a;
    memset(&a, 0, sizeof a);
    if (int rc = check_cache(c, scales, t, &a.c)) return rc;
    if (int rc = check_count(R)) return rc;
    if (tokens < 1 || tokens > 65536 || R % tokens) return bad("tokens must be 1..65536, a divisor of the rows");
    if (window < 0 || window > kMaxLen || sink < 0 || sink > kMaxLen) return bad("window and sink must be 0..2^30");
    if (sink && !window) return bad("sink without a window");
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
    // (its kernel counts the workgroups of all heads in one int)
    const int64_t tiles = (q_heads / c->kv_heads + 15) / 16;
    if (c->dtype == XT_I8 && R * c->kv_heads * tiles > kMaxInt)
        return bad("rows times key-value heads (a head for every 16 query heads) must be below 2^31");
    set_scales(scales, &a);
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
    a.window = (int)(window ? window : kMaxLen);
    a.sink = (int)sink;
    a.tokens = (int)tokens;
    int64_t part = R;  // rows at a time
    if (a.accumulate) {
        // (a table that no device holds a row's scores of is refused, whatever the
        // window; a row's scores are those of the positions that it may see.  Every
        // row makes its own pass, so parts need not be whole groups.)
        const int64_t cap = t->max_pages * c->page_size, seen = std::min(cap, (int64_t)a.window + a.sink);
        if (int rc = check_fits(4.0 * q_heads * (double)cap, "the workspace")) return rc;
        part = part_of(R, 4 * (int64_t)q_heads * seen);
    }
    int cus = 0;
    if (int rc = xt_internal_cus(&cus)) return rc;
    hipStream_t st = static_cast<hipStream_t>(stream);
    void *ws, *counters;
    size_t nc, nc_last;
    const xt::AttnArgs last = rows_of(a, (R - 1) / part * part, R - (R - 1) / part * part);
    const bool codes = c->dtype == XT_I8;
    const auto workspace = codes ? xt::attention8_workspace : xt::attention_workspace;
    const size_t bytes_last = workspace(last, cus, &nc_last);
    const size_t bytes = std::max(bytes_last, workspace(rows_of(a, 0, part), cus, &nc));
    if (int rc = get_workspace(st, bytes, std::max(nc, nc_last), &ws, &counters)) return rc;
    for (int64_t r0 = 0; r0 < R; r0 += part) {
        const xt::AttnArgs b = rows_of(a, r0, std::min(part, R - r0));
        const hipError_t e = codes ? xt::launch_paged_attention8(b, cus, ws, counters, st)
                                   : xt::launch_paged_attention(c->dtype, b, cus, ws, counters, st);
        if (int rc = launched(e, "paged attention launch")) return rc;
    }
    return XT_OK;
}

int xt_kv_evict(const xt_kv_cache* c, const xt_kv_table* t, const int32_t* lengths, int64_t budget, int64_t sink,
                int64_t recent, int32_t* new_lengths, int32_t* kept, void* stream) {
    xt::EvictArgs a;
    memset(&a, 0, sizeof a);
    if (c && c->dtype == XT_I8) return bad("eviction needs a cache with scores, which one of 8-bit codes does not keep");
    if (int rc = check_cache(c, nullptr, t, &a.c)) return rc;
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

int xt_verify_drafts(int dtype, const void* target, int64_t ld_seq, int64_t ld_row, const void* draft, int64_t ldd_seq,
                     int64_t ldd_row, int64_t S, int64_t T, int64_t V, const int32_t* drafted, const int32_t* counts,
                     const float* uniforms, float temperature, const float* temperatures, int32_t* accepted,
                     int32_t* tokens, float* logprobs, void* stream) {
    if (int rc = check_dtype(dtype)) return rc;
    if (T < 0 || T > xt::kVerifyDrafts) return bad("drafts of a sequence must be 0..64");
    if (S < 0 || S > kMaxRows || S * (2 * T + 1) > kMaxRows) return bad("sequences times 2 drafts + 1 must be 0..2^21");
    if (V < 1 || V > (1 << 30)) return bad("vocabulary must be 1..2^30");
    if (!temperatures && !(temperature >= 0.0f && isfinite(temperature))) return bad("temperature must be finite, >= 0");
    if (S == 0) return XT_OK;
    if (!target || !uniforms || !accepted || !tokens || !logprobs || (T > 0 && !drafted)) return bad("NULL pointer");
    const int es = dtype == XT_F32 ? 4 : 2;
    if (int rc = check_logits(target, ld_seq, ld_row, S, T + 1, V, "target", es)) return rc;
    if (draft && T > 0) {
        if (int rc = check_logits(draft, ldd_seq, ldd_row, S, T, V, "draft", es)) return rc;
    }
    struct Words {
        const void* p;
        int64_t n;  // words
        const char* what;
    };
    const Words words[] = {{drafted, S * T, "drafted"},   {counts, S, "counts"},           {uniforms, S * (T + 1), "uniforms"},
                 {temperatures, S, "temperatures"}, {accepted, S, "accepted"}, {tokens, S * (T + 1), "tokens"},
                 {logprobs, S * (T + 1), "logprobs"}};
    for (const auto& w : words)
        if (int rc = check_align(w.p, 4, w.what)) return rc;
    // (a sequence's workgroups read the inputs at any time before its last one
    // writes, and those of one that ends early after that, too)
    for (int i = 4; i < 7; ++i)
        for (int j = 0; j < i; ++j) {
            const uintptr_t x = reinterpret_cast<uintptr_t>(words[i].p), y = reinterpret_cast<uintptr_t>(words[j].p);
            if (y && x < y + 4 * (uintptr_t)words[j].n && y < x + 4 * (uintptr_t)words[i].n)
                return bad(std::string(words[i].what) + " overlaps " + words[j].what);
        }
    for (int i = 4; i < 7; ++i) {
        const Words& w = words[i];
        const uintptr_t x = reinterpret_cast<uintptr_t>(w.p);
        if (meets_logits(x, 4 * (uint64_t)w.n, target, ld_seq, ld_row, S, T + 1, V, es))
            return bad(std::string(w.what) + " overlaps target");
        if (draft && T > 0 && meets_logits(x, 4 * (uint64_t)w.n, draft, ldd_seq, ldd_row, S, T, V, es))
            return bad(std::string(w.what) + " overlaps draft");
    }
    xt::VerifyArgs a;
    memset(&a, 0, sizeof a);
    a.target = target;
    a.draft = T > 0 ? draft : nullptr;
    a.ld_seq = S > 1 ? ld_seq : 0;
    a.ld_row = T > 0 ? ld_row : 0;
    a.ldd_seq = S > 1 ? ldd_seq : 0;
    a.ldd_row = T > 1 ? ldd_row : 0;
    a.S = (int)S;
    a.T = (int)T;
    a.V = (int)V;
    a.drafted = drafted;
    a.counts = counts;
    a.uniforms = uniforms;
    a.temps = temperatures;
    a.temp = temperature;
    a.accepted = accepted;
    a.tokens = tokens;
    a.logprobs = logprobs;
    int cus = 0;
    if (int rc = xt_internal_cus(&cus)) return rc;
    hipStream_t st = static_cast<hipStream_t>(stream);
    void *ws, *counters;
    size_t nc;
    const size_t bytes = xt::verify_workspace(a, cus, &nc);
    if (int rc = get_workspace(st, bytes, nc, &ws, &counters)) return rc;
    return launched(xt::launch_verify(dtype, a, cus, ws, counters, st), "draft verification launch");
}

}  // extern "C"
