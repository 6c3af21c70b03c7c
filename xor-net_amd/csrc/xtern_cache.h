// Internal declarations of the paged key-value cache (append, read-back,
// attention, eviction), of the token probabilities and of the verification of
// drafted tokens: kernel arguments and launchers (xtern_attn.hip,
// xtern_attn8.hip, xtern_store.hip, xtern_evict.hip, xtern_probs.hip,
// xtern_verify.hip), called by xtern_cache_api.cpp.
#pragma once
#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "../../include/xtern.h"

namespace xt {

// n / d for n < 2^31 as n * mul >> shift: mul = ceil(2^(31 + s) / d), shift =
// 31 + s, 2^s >= d (d <= 65536); the error of mul, below d <= 2^s, grows to
// less than 2^(31 + s) in the product.
struct FastDiv {
    unsigned mul;
    int shift;
};
inline FastDiv fast_div(int d) {
    int s = 0;
    while ((1 << s) < d) ++s;
    return FastDiv{(unsigned)((((uint64_t)1 << (31 + s)) + (uint64_t)d - 1) / (uint64_t)d), 31 + s};
}

// The cache as the kernels see it: strides in elements, score
// [num_pages][hkv][page] or null.  (What only some calls have stands at the end of
// their arguments: a line of these more that the others' kernels wait for is 0.04
// us of an append's 3.)
struct KvView {
    void* k;
    void* v;
    float* score;
    int64_t sp, ss, sh;  // element strides of a page, a slot, a head
    int num_pages, page, hkv, D;
    FastDiv by_page;
    const int32_t* table;  // [nseq][max_pages], row stride ldt
    int64_t ldt;
    int nseq, max_pages;
};

struct AppendArgs {
    KvView c;
    const int32_t* seq;    // [R] or null (row r belongs to sequence r)
    const int32_t* slots;  // [R] cache positions; negative: no row
    const int32_t* pos;    // [R] rotary positions (rope only)
    const float* cos;      // [rope_rows][rot / 2], or null (no rotation)
    const float* sin;
    int64_t rope_rows;
    int rot;
    const float* q;        // [R] rows of hq * D, stride ldq; or null
    float* qo;
    const float* k;
    const float* v;
    int32_t* lengths;      // [R] or null: positions that the row's token sees, 0 for a skipped row
    int64_t ldq, ldqo, ldk, ldv;
    int hq;
    int64_t R;
    FastDiv by_per, by_vals;  // set by the launcher
    const float* q_norm;      // [D] weights of a head's norm, or null (no norms)
    const float* k_norm;
    double eps;
    double inv_dim;           // 1 / D, set by the launcher
    float* ks;                // 8-bit codes: the scales [num_pages][hkv][page] of keys and of values
    float* vs;
};
hipError_t launch_kv_append(int dtype, AppendArgs a, hipStream_t s);
// With norms, or into 8-bit codes; cus: compute units of the device.
hipError_t launch_kv_store(int dtype, AppendArgs a, int cus, hipStream_t s);

struct ReadArgs {
    KvView c;
    const int32_t* seq;    // [R] or null
    const int32_t* slots;  // [R]
    void* k;               // [R] rows of hkv * D, strides ldk, ldv
    void* v;
    int64_t ldk, ldv;
    int64_t R;
    FastDiv by_per;        // set by the launcher
    const float* ks;       // as above
    const float* vs;
};
hipError_t launch_kv_read(int dtype, int out, ReadArgs a, int cus, hipStream_t s);

struct AttnArgs {
    KvView c;
    const int32_t* seq;      // [R] or null
    const int32_t* lengths;  // [R]
    const float* q;
    float* out;
    float* lse;              // [R][hq] or null
    int64_t ldq, ldo;
    int hq;
    float scale;
    int accumulate;
    int64_t R;
    int64_t call_rows;       // of the call whose rows, or a part of them, these are
    int window, sink;        // a row of length n sees p < sink and p >= n - window (2^30: every p)
    int tokens;              // rows r of one sequence: (row0 + r) / tokens, numbered as
                             // seq and the table are (of the whole call where tokens > 1)
    int row0;
    // set by the launcher: a sequence's rows, in units of unit_rows
    int unit_rows, units;
    FastDiv by_units;
    const float* ks;         // as above
    const float* vs;
};
// Bytes of workspace that the call needs, and of counters that are zero before
// and after it (0: none, null); cus: compute units of the device.
size_t attention_workspace(const AttnArgs& a, int cus, size_t* counters);
hipError_t launch_paged_attention(int dtype, AttnArgs a, int cus, void* ws, void* counters, hipStream_t s);
// The same over a cache of 8-bit codes.
size_t attention8_workspace(const AttnArgs& a, int cus, size_t* counters);
hipError_t launch_paged_attention8(AttnArgs a, int cus, void* ws, void* counters, hipStream_t s);

struct EvictArgs {
    KvView c;
    const int32_t* lengths;  // [nseq]
    int32_t* new_lengths;    // [nseq]
    int32_t* kept;           // [nseq][hkv][budget]
    int budget, sink, recent;
    // workspace (set by the launcher): keys [nseq][hkv][ldk], staged rows
    unsigned* keys;
    int64_t ldk;
    int __attribute__((ext_vector_type(4)))* stage;
    float* stage_score;
};
// Bytes of keys in it for each sequence; the whole of it.
size_t evict_key_bytes(const EvictArgs& a);
size_t evict_workspace(int dtype, const EvictArgs& a, int cus);
hipError_t launch_kv_evict(int dtype, EvictArgs a, int cus, void* ws, hipStream_t s);

struct ProbsArgs {
    const void* x;  // [M] rows of V logits, stride ld
    int64_t ld;
    int64_t M;
    int V;
    const int32_t* tokens;  // [M][T]
    int T;
    float* lp;       // [M][T]
    float* entropy;  // [M]
    int top;
    int32_t* ids;    // [M][top]
    float* top_lp;   // [M][top]
};
size_t token_logprobs_workspace(const ProbsArgs& a, int cus, size_t* counters);
hipError_t launch_token_logprobs(int dtype, const ProbsArgs& a, int cus, void* ws, void* counters, hipStream_t s);

constexpr int kVerifyDrafts = 64;  // of a sequence: a lane each

struct VerifyArgs {
    const void* target;  // [S][T + 1][V], strides in elements
    const void* draft;   // [S][T][V] or null
    int64_t ld_seq, ld_row, ldd_seq, ldd_row;
    int S, T, V;
    const int32_t* drafted;  // [S][T]
    const int32_t* counts;   // [S] or null
    const float* uniforms;   // [S][T + 1]
    const float* temps;      // [S] or null
    float temp;
    int32_t* accepted;       // [S]
    int32_t* tokens;         // [S][T + 1]
    float* logprobs;         // [S][T + 1]
};
size_t verify_workspace(const VerifyArgs& a, int cus, size_t* counters);
hipError_t launch_verify(int dtype, const VerifyArgs& a, int cus, void* ws, void* counters, hipStream_t s);

#ifdef __HIPCC__
}  // namespace xt
#include "xtern_device.h"
namespace xt {

// Inclusive sum over the wave's lanes.
__device__ __forceinline__ int wave_scan(int v) {
    v += dpp_id<0x111, 0xf>(v);
    v += dpp_id<0x112, 0xf>(v);
    v += dpp_id<0x114, 0xf>(v);
    v += dpp_id<0x118, 0xf>(v);
    v += dpp_id<0x142, 0xa>(v);
    v += dpp_id<0x143, 0xc>(v);
    return v;
}

// Counts bin `bin` of a histogram in LDS for every lane that is `in`: one add
// for a wave whose lanes agree (a tile of equal values would otherwise add to
// one address lane by lane).
__device__ __forceinline__ void hist_add(int* hist, int bin, bool in) {
    const unsigned long long who = __ballot(in);
    if (!who) return;
    const int first = __builtin_ctzll(who), b = __builtin_amdgcn_readlane(bin, first);
    if (__ballot(in && bin == b) == who) {
        if ((int)(threadIdx.x & 63) == first) atomicAdd(&hist[b], (int)__popcll(who));
    } else if (in) {
        atomicAdd(&hist[bin], 1);
    }
}

// Of a 256-bin histogram in LDS, by every wave for itself: the highest bin b
// such that bins b .. 255 hold at least `need`; *left = what b has to give.
// One step of finding the need-th largest of many 32-bit keys, 8 bits a pass.
__device__ __forceinline__ int radix_bin(const int* hist, int need, int* left) {
    const int lane = threadIdx.x & 63;
    int c[4], sum = 0;  // lane l: bins 255 - 4 l downwards
    for (int i = 0; i < 4; ++i) sum += c[i] = hist[255 - 4 * lane - i];
    const int upto = wave_scan(sum);
    const int l = __builtin_ctzll(__ballot(upto >= need));
    int before = upto - sum, i = 0;
    while (i < 3 && before + c[i] < need) before += c[i++];
    *left = __builtin_amdgcn_readlane(need - before, l);
    return __builtin_amdgcn_readlane(255 - 4 * lane - i, l);
}

// One element of the cache or of the logits as f32, and back (round to
// nearest even; f16 overflows to infinity).
template <int DT> struct Elem;
template <> struct Elem<XT_F32> {
    typedef float T;
    static __device__ __forceinline__ float get(T v) { return v; }
    static __device__ __forceinline__ T put(float v) { return v; }
};
template <> struct Elem<XT_F16> {
    typedef _Float16 T;
    static __device__ __forceinline__ float get(T v) { return (float)v; }
    static __device__ __forceinline__ T put(float v) { return (T)v; }
};
template <> struct Elem<XT_BF16> {
    typedef __bf16 T;
    static __device__ __forceinline__ float get(T v) { return (float)v; }
    static __device__ __forceinline__ T put(float v) { return (T)v; }
};

__device__ __forceinline__ int fast_quot(int n, FastDiv d) {
    return (int)(((uint64_t)(unsigned)n * d.mul) >> d.shift);
}
__device__ __forceinline__ int kv_page_of(const KvView& c, int p) { return fast_quot(p, c.by_page); }
// The page that holds position p of sequence `seq`, or -1: a table entry
// outside the pool holds nothing.  0 <= p < max_pages * page.
__device__ __forceinline__ int kv_page(const KvView& c, int seq, int p) {
    const int e = c.table[(int64_t)seq * c.ldt + kv_page_of(c, p)];
    return (unsigned)e < (unsigned)c.num_pages ? e : -1;
}
// Its slot there.
__device__ __forceinline__ int kv_slot(const KvView& c, int p) { return p - kv_page_of(c, p) * c.page; }
__device__ __forceinline__ int64_t kv_offset(const KvView& c, int pg, int p, int h) {
    return (int64_t)pg * c.sp + (int64_t)kv_slot(c, p) * c.ss + (int64_t)h * c.sh;
}
// A length as the kernels use it: within the table's row.
__device__ __forceinline__ int kv_length(const KvView& c, int n) {
    const int64_t cap = (int64_t)c.max_pages * c.page;
    return n < 0 ? 0 : (n > cap ? (int)cap : n);
}

#endif

}  // namespace xt
