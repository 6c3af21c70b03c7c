// Eviction from the paged key-value cache by accumulated attention weight.
//
// Per sequence of n > budget positions and per key-value head: the first
// `sink` and the last `recent` positions stay, and of those between the
// `need` = budget - sink - recent of the highest score (ties to the lowest
// position; NaN below every number, a position without a page below that).
// They move, in order, to positions 0 .. budget - 1.
//
// One workgroup per (sequence, head).  Selection: the need-th highest 32-bit
// key by four passes of an 8-bit histogram, then one pass in position order
// that writes the kept list.  Moving in place: the kept list is ascending, so
// kept[j] >= j, and a chunk of targets j0 .. j1 - 1 never holds a source of a
// later chunk; inside a chunk every load comes before the first store.
#include "xtern_cache.h"
#include "xtern_device.h"

namespace xt {

constexpr int kEvictThreads = 1024;
constexpr int kEvictWaves = kEvictThreads / 64;

__device__ __forceinline__ unsigned evict_key(const KvView& c, int seq, int h, int p) {
    const int pg = kv_page(c, seq, p);
    if (pg < 0) return 0u;
    const float f = c.score[((int64_t)pg * c.hkv + h) * c.page + p % c.page] + 0.0f;  // (-0 counts as +0)
    if (f != f) return 1u;
    const unsigned u = __float_as_uint(f);
    return u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u);
}

// Copies rows of `units` T from position kept[j] to j for the j whose
// position changes.
template <typename T>
__device__ void move_rows(const KvView& c, int seq, int h, T* base, int64_t sp, int64_t ss, int64_t sh,
                          int units, const int32_t* kept, int j0, int budget) {
    const int64_t total = (int64_t)(budget - j0) * units;
    for (int64_t i0 = 0; i0 < total; i0 += kEvictThreads) {
        const int64_t i = i0 + threadIdx.x;
        T val{};
        int64_t to = -1;
        if (i < total) {
            const int j = j0 + (int)(i / units), u = (int)(i % units), src = kept[j];
            const int pf = kv_page(c, seq, src), pt = kv_page(c, seq, j);
            if (src != j && pf >= 0 && pt >= 0) {
                val = base[pf * sp + (src % c.page) * ss + h * sh + u];
                to = pt * sp + (j % c.page) * ss + h * sh + u;
            }
        }
        __syncthreads();
        if (to >= 0) base[to] = val;
        __syncthreads();
    }
}

template <typename T>
__global__ __launch_bounds__(kEvictThreads) void kv_evict_kernel(EvictArgs a, int per_unit) {
    const KvView& c = a.c;
    const int seq = blockIdx.x, h = blockIdx.y, t = threadIdx.x, wave = t >> 6, lane = t & 63;
    __shared__ int hist[256];
    __shared__ int wcount[2][kEvictWaves];
    __shared__ int pick[2];
    const int n = kv_length(c, a.lengths[seq]);
    int32_t* kept = a.kept + ((int64_t)seq * c.hkv + h) * a.budget;
    if (h == 0 && t == 0) a.new_lengths[seq] = min(n, a.budget);
    if (n <= a.budget) {
        for (int j = t; j < a.budget; j += kEvictThreads) kept[j] = j < n ? j : -1;
        return;
    }
    const int lo = a.sink, hi = n - a.recent;  // the positions between
    int need = a.budget - a.sink - a.recent;
    unsigned prefix = 0;
    if (need > 0) {
        for (int shift = 24; shift >= 0; shift -= 8) {
            if (t < 256) hist[t] = 0;
            __syncthreads();
            const unsigned mask = shift == 24 ? 0u : ~0u << (shift + 8);
            for (int p = lo + t; p < hi; p += kEvictThreads) {
                const unsigned k = evict_key(c, seq, h, p);
                if ((k & mask) == prefix) atomicAdd(&hist[(k >> shift) & 255], 1);
            }
            __syncthreads();
            if (t == 0) {
                int left = need, b = 255;
                while (hist[b] < left) left -= hist[b--];
                pick[0] = b;
                pick[1] = left;
            }
            __syncthreads();
            prefix |= (unsigned)pick[0] << shift;
            need = pick[1];  // of the keys equal to the prefix so far, as many stay
        }
    }
    // kept: keys above `prefix`, and the first `need` equal to it
    const bool any = a.budget > a.sink + a.recent;
    const int per = ((hi - lo + kEvictWaves - 1) / kEvictWaves + 63) / 64 * 64;
    const int w0 = lo + wave * per, w1 = min(w0 + per, hi);
    int above = 0, equal = 0;
    if (any)
        for (int p = w0; p < w1; p += 64) {
            const unsigned k = p + lane < w1 ? evict_key(c, seq, h, p + lane) : 0u;
            above += __popcll(__ballot(p + lane < w1 && k > prefix));
            equal += __popcll(__ballot(p + lane < w1 && k == prefix));
        }
    if (lane == 0) {
        wcount[0][wave] = above;
        wcount[1][wave] = equal;
    }
    for (int j = t; j < a.sink; j += kEvictThreads) kept[j] = j;
    for (int j = t; j < a.recent; j += kEvictThreads) kept[a.budget - a.recent + j] = hi + j;
    __syncthreads();
    if (any) {
        int eq = 0, at = a.sink;
        for (int w = 0; w < wave; ++w) {
            const int e = min(wcount[1][w], max(0, need - eq));
            eq += wcount[1][w];
            at += wcount[0][w] + e;
        }
        const unsigned long long below = (1ull << lane) - 1;
        for (int p = w0; p < w1; p += 64) {
            const bool in = p + lane < w1;
            const unsigned k = in ? evict_key(c, seq, h, p + lane) : 0u;
            const unsigned long long me = __ballot(in && k == prefix);
            const bool take = in && (k > prefix || (k == prefix && eq + __popcll(me & below) < need));
            const unsigned long long mt = __ballot(take);
            if (take) kept[at + __popcll(mt & below)] = p + lane;
            eq += __popcll(me);
            at += __popcll(mt);
        }
    }
    __syncthreads();
    const int units = c.D / per_unit;
    move_rows<T>(c, seq, h, static_cast<T*>(c.k), c.sp / per_unit, c.ss / per_unit, c.sh / per_unit, units, kept,
                 a.sink, a.budget);
    move_rows<T>(c, seq, h, static_cast<T*>(c.v), c.sp / per_unit, c.ss / per_unit, c.sh / per_unit, units, kept,
                 a.sink, a.budget);
    move_rows<float>(c, seq, h, c.score, (int64_t)c.hkv * c.page, 1, c.page, 1, kept, a.sink, a.budget);
}

hipError_t launch_kv_evict(int dtype, const EvictArgs& a, hipStream_t s) {
    const KvView& c = a.c;
    const int es = dtype == XT_F32 ? 4 : 2;
    // the widest unit that every row starts and ends on
    const uint64_t bits = (uint64_t)reinterpret_cast<uintptr_t>(c.k) | (uint64_t)reinterpret_cast<uintptr_t>(c.v) |
                          (uint64_t)(c.sp * es) | (uint64_t)(c.ss * es) | (uint64_t)(c.sh * es) | (uint64_t)(c.D * es);
    const dim3 grid((unsigned)c.nseq, (unsigned)c.hkv), block(kEvictThreads);
    if (!(bits & 15))
        kv_evict_kernel<v4i><<<grid, block, 0, s>>>(a, 16 / es);
    else if (!(bits & 3))
        kv_evict_kernel<int><<<grid, block, 0, s>>>(a, 4 / es);
    else
        kv_evict_kernel<short><<<grid, block, 0, s>>>(a, 1);
    return hipGetLastError();
}

}  // namespace xt
