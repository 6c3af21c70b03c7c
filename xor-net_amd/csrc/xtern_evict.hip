// Eviction from the paged key-value cache by accumulated attention weight.
//
// Per sequence of n > budget positions and per key-value head, of the
// positions that have a page, L[0] < L[1] < ..: the first `sink` and the last
// `recent` stay, and of those between the `need` = budget - sink - recent of
// the highest score (ties to the lowest position; NaN below every number).
// The j-th that stays moves to L[j].  Where no page is missing L[j] = j, which
// is what the fast paths take (to look for missing pages costs the selection
// 0.4 us); a workgroup that meets one takes its L from the table, a stretch of
// entries at a time.
//
// First the selection, one workgroup per (sequence, head): the scores as
// 32-bit keys, the need-th highest by four passes of an 8-bit histogram, then
// the kept list in position order.  Up to 16384 positions the keys stay in
// registers; for more, a kernel of its own writes them to a workspace first
// (finding a score takes forty instructions, reading a key a few: 40000
// positions of 8 heads 8 + 48 us, 80 with the selecting workgroup finding its own).
// Then the moving: HBM bounds it (every kept row is read and written once); a
// workgroup per (sequence, head, tensor), and per part of a row where those
// are too few for the chip.  32 sequences of up to 8192 positions and 8 heads
// of 128 in f16, cut to 2048: 17 + 95 us (4.3 TB/s moved; a large copy reaches
// 4.8); one of 1027 positions and 5 heads cut to 512: 10 + 6 us.
//
// Why rows can move in place: the kept list ascends and is part of L, so
// kept[j] >= L[j].  A workgroup moves its part of the rows in rounds of
// ascending j.  A source of a later round is never the target of an earlier
// one (it is no lower than its own L[j], which is above every earlier one), so a round needs no earlier
// store to be done; and a target is a source only of its own or an earlier
// round, so the barrier between a round's loads and its stores is enough.
#include <algorithm>
#include <type_traits>

#include "xtern_cache.h"

namespace xt {

constexpr int kEvictThreads = 1024;
constexpr int kEvictWaves = kEvictThreads / 64;
constexpr int kEvictRegs = 16;  // keys of a thread that stay in registers
constexpr int kMoveUnits = 4;   // 16-byte pieces of a thread and round
constexpr int kEvictAhead = 8;  // keys of a thread in flight where they go through memory
constexpr int kEvictTile = 256 * kEvictAhead;

__device__ __forceinline__ unsigned evict_key(const KvView& c, int seq, int h, int p) {
    const int pg = kv_page(c, seq, p);
    if (pg < 0) return 0u;
    const float f = c.score[((int64_t)pg * c.hkv + h) * c.page + kv_slot(c, p)] + 0.0f;  // (-0 counts as +0)
    if (f != f) return 1u;
    const unsigned u = __float_as_uint(f);
    return u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u);
}

// The next THREADS entries of a sequence's table from `at` on, below `pages`:
// those that are a page, in order, to list; returns how many.  By the whole
// workgroup; list [THREADS], counts [THREADS / 64] in LDS.
template <int THREADS>
__device__ __forceinline__ int live_entries(const KvView& c, int seq, int pages, int at, int* list, int* counts) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i = at + (int)threadIdx.x;
    const int e = i < pages ? c.table[(int64_t)seq * c.ldt + i] : -1;
    const bool live = (unsigned)e < (unsigned)c.num_pages;
    const unsigned long long who = __ballot(live);
    __syncthreads();  // (the list before may still be read)
    if (lane == 0) counts[wave] = (int)__popcll(who);
    __syncthreads();
    int before = 0, total = 0;
    for (int w = 0; w < THREADS / 64; ++w) {
        if (w < wave) before += counts[w];
        total += counts[w];
    }
    if (live) list[before + (int)__popcll(who & ((1ull << lane) - 1))] = i;
    __syncthreads();
    return total;
}
__device__ __forceinline__ int kv_pages(const KvView& c, int n) { return n > 0 ? kv_page_of(c, n - 1) + 1 : 0; }

// Keys of the positions between, to the workspace, by the whole chip: for
// calls whose heads may have more than a workgroup's registers hold.
__global__ __launch_bounds__(256) void kv_evict_keys_kernel(EvictArgs a) {
    const KvView& c = a.c;
    const int seq = blockIdx.x, h = blockIdx.y, n = kv_length(c, a.lengths[seq]);
    const int mid = n - a.recent - a.sink;
    if (n <= a.budget || mid <= kEvictRegs * kEvictThreads) return;
    unsigned* keys = a.keys + ((int64_t)seq * c.hkv + h) * a.ldk;
    for (int64_t p0 = (int64_t)blockIdx.z * kEvictTile + threadIdx.x; p0 < mid; p0 += (int64_t)gridDim.z * kEvictTile) {
        unsigned k[kEvictAhead];
#pragma unroll
        for (int i = 0; i < kEvictAhead; ++i)
            k[i] = evict_key(c, seq, h, a.sink + (int)min(p0 + 256 * i, (int64_t)mid - 1));
#pragma unroll
        for (int i = 0; i < kEvictAhead; ++i)
            if (p0 + 256 * i < mid) keys[p0 + 256 * i] = k[i];
    }
}

__global__ __launch_bounds__(kEvictThreads) void kv_evict_select_kernel(EvictArgs a) {
    const KvView& c = a.c;
    const int seq = blockIdx.x, h = blockIdx.y, t = threadIdx.x, wave = t >> 6, lane = t & 63;
    __shared__ int hist[4][256];
    __shared__ int count[2][kEvictRegs * kEvictWaves];  // above and equal, by chunk of 64 positions
    __shared__ bool wave_missing[kEvictWaves];
    __shared__ int between[2];  // tables with missing pages: the positions that end `sink` and begin `recent`
    const int n = kv_length(c, a.lengths[seq]);
    int32_t* kept = a.kept + ((int64_t)seq * c.hkv + h) * a.budget;
    if (n <= a.budget) {
        if (h == 0 && t == 0) a.new_lengths[seq] = n;
        for (unsigned j = t; j < (unsigned)a.budget; j += kEvictThreads)  // (up to 2^31 - 1)
            kept[j] = (int)j < n ? (int)j : -1;
        return;
    }
    int lo = a.sink, hi = n - a.recent, mid = hi - lo;  // the positions between
    int need = a.budget - a.sink - a.recent;
    bool regs = mid <= kEvictRegs * kEvictThreads;
    unsigned* keys = a.keys + ((int64_t)seq * c.hkv + h) * a.ldk;  // (where they do not fit)
    int used;                  // registers in use
    unsigned key[kEvictRegs];  // position lo + 1024 i + t
    auto load_keys = [&]() {
        used = regs && need ? (mid + kEvictThreads - 1) / kEvictThreads : 0;
#pragma unroll
        for (int i = 0; i < kEvictRegs; ++i) {
            const int p = lo + i * kEvictThreads + t;
            key[i] = 0u;
            if (i < used && p < hi) key[i] = evict_key(c, seq, h, p);
        }
    };
    load_keys();
    // Pages that are missing (with the keys' loads in flight)
    const int pages = kv_pages(c, n);
    bool missing = false;
    for (int p = t; p < pages; p += kEvictAhead * kEvictThreads) {
        int e[kEvictAhead];
#pragma unroll
        for (int i = 0; i < kEvictAhead; ++i)
            e[i] = c.table[(int64_t)seq * c.ldt + min(p + i * kEvictThreads, pages - 1)];
#pragma unroll
        for (int i = 0; i < kEvictAhead; ++i) missing |= (unsigned)e[i] >= (unsigned)c.num_pages;
    }
    if (t < 256)
        for (int i = 0; i < 4; ++i) hist[i][t] = 0;
    missing = __any(missing);
    if (lane == 0) wave_missing[wave] = missing;
    __syncthreads();
    if (!__any(wave_missing[lane % kEvictWaves])) {
        if (h == 0 && t == 0) a.new_lengths[seq] = a.budget;
        for (int j = t; j < a.sink; j += kEvictThreads) kept[j] = j;
        for (int j = t; j < a.recent; j += kEvictThreads) kept[a.budget - a.recent + j] = hi + j;
    } else {
        // (the lists in what the histograms and counts take later)
        int *list = hist[0], *counts = count[0];
        int entries = 0, live = 0;
        for (int at = 0; at < pages; at += kEvictThreads)
            entries += live_entries<kEvictThreads>(c, seq, pages, at, list, counts);
        live = entries * c.page;
        const int tail = c.table[(int64_t)seq * c.ldt + pages - 1];
        if ((unsigned)tail < (unsigned)c.num_pages) live -= pages * c.page - n;
        const int stay = min(live, a.budget);
        const bool all = live <= a.budget;
        if (t == 0 && all && h == 0 && live == 0) a.new_lengths[seq] = 0;
        for (int j = live + t; j < a.budget; j += kEvictThreads) kept[j] = -1;
        int before = 0;  // entries before the list's
        for (int at = 0; at < pages; at += kEvictThreads) {
            const int m = live_entries<kEvictThreads>(c, seq, pages, at, list, counts);
            for (int x = t; x < m * c.page; x += kEvictThreads) {
                const int e = kv_page_of(c, x), p = list[e] * c.page + x - e * c.page, j = before * c.page + x;
                if (p >= n) continue;  // p = L[j]
                if (all || j < a.sink) kept[j] = p;
                else if (j >= live - a.recent) kept[j - live + a.budget] = p;
                if (j == a.sink) between[0] = p;
                if (j == live - a.recent) between[1] = p;
                if (j == stay - 1 && h == 0) a.new_lengths[seq] = p + 1;
            }
            before += m;
        }
        if (all) return;
        __syncthreads();
        // the positions between, holes among them: their keys, 0, are below
        // every other, and there are more than `need` of the others
        lo = between[0];
        hi = a.recent ? between[1] : n;
        mid = hi - lo;
        keys += lo - a.sink;
        regs = mid <= kEvictRegs * kEvictThreads;
        load_keys();
        for (int i = t; i < 4 * 256; i += kEvictThreads) list[i] = 0;
        __syncthreads();
    }
    if (need == 0) return;
    unsigned prefix = 0;
    for (int pass = 0; pass < 4; ++pass) {
        const int shift = 24 - 8 * pass;
        const unsigned mask = pass ? ~0u << (shift + 8) : 0u;
        if (regs) {
#pragma unroll
            for (int i = 0; i < kEvictRegs; ++i)
                if (i < used)
                    hist_add(hist[pass], (key[i] >> shift) & 255,
                             lo + i * kEvictThreads + t < hi && (key[i] & mask) == prefix);
        } else {
            for (int p = t; p < mid; p += kEvictAhead * kEvictThreads) {
                unsigned k[kEvictAhead];
#pragma unroll
                for (int i = 0; i < kEvictAhead; ++i) k[i] = keys[min(p + i * kEvictThreads, mid - 1)];
#pragma unroll
                for (int i = 0; i < kEvictAhead; ++i) {
                    const bool in = p + i * kEvictThreads < mid;
                    hist_add(hist[pass], (k[i] >> shift) & 255, in && (k[i] & mask) == prefix);
                }
            }
        }
        __syncthreads();
        int left;
        prefix |= (unsigned)radix_bin(hist[pass], need, &left) << shift;
        need = left;  // of the keys equal to the prefix so far, as many stay
    }
    // kept: keys above `prefix`, and the first `need` equal to it
    const unsigned long long below = (1ull << lane) - 1;
    const int at0 = a.sink;
    if (regs) {
#pragma unroll
        for (int i = 0; i < kEvictRegs; ++i) {
            if (i >= used) {
                if (lane == 0) count[0][i * kEvictWaves + wave] = count[1][i * kEvictWaves + wave] = 0;
                continue;
            }
            const bool in = lo + i * kEvictThreads + t < hi;
            const int above = __popcll(__ballot(in && key[i] > prefix));
            const int equal = __popcll(__ballot(in && key[i] == prefix));
            if (lane == 0) {
                count[0][i * kEvictWaves + wave] = above;
                count[1][i * kEvictWaves + wave] = equal;
            }
        }
        __syncthreads();
        // sums before each chunk: wave 0 the ones above, wave 1 the equal ones
        if (wave < 2) {
            int* cnt = count[wave] + 4 * lane;
            int v[4], sum = 0;
            for (int i = 0; i < 4; ++i) sum += v[i] = cnt[i];
            int before = wave_scan(sum) - sum;
            for (int i = 0; i < 4; ++i) {
                cnt[i] = before;
                before += v[i];
            }
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kEvictRegs; ++i) {
            if (i >= used) continue;
            const int p = lo + i * kEvictThreads + t;
            const int eq = count[1][i * kEvictWaves + wave];
            const unsigned long long me = __ballot(p < hi && key[i] == prefix);
            const bool take = p < hi && (key[i] > prefix || (key[i] == prefix && eq + __popcll(me & below) < need));
            const unsigned long long mt = __ballot(take);
            if (take) kept[at0 + count[0][i * kEvictWaves + wave] + min(eq, need) + __popcll(mt & below)] = p;
        }
        return;
    }
    // a stretch of positions per wave, counted and then written
    const int per = ((mid + kEvictWaves - 1) / kEvictWaves + 63) / 64 * 64;
    const int w0 = (int)min((int64_t)lo + (int64_t)wave * per, (int64_t)hi), w1 = min(w0 + per, hi);
    int above = 0, equal = 0;
    for (int p = w0; p < w1; p += 64 * kEvictAhead) {
        unsigned k[kEvictAhead];
#pragma unroll
        for (int i = 0; i < kEvictAhead; ++i) k[i] = keys[min(p + 64 * i + lane, hi - 1) - lo];
#pragma unroll
        for (int i = 0; i < kEvictAhead; ++i) {
            const bool in = p + 64 * i + lane < w1;
            above += __popcll(__ballot(in && k[i] > prefix));
            equal += __popcll(__ballot(in && k[i] == prefix));
        }
    }
    if (lane == 0) {
        count[0][wave] = above;
        count[1][wave] = equal;
    }
    __syncthreads();
    int eq = 0, at = at0;
    for (int w = 0; w < wave; ++w) {
        at += count[0][w] + min(count[1][w], max(0, need - eq));
        eq += count[1][w];
    }
    for (int p = w0; p < w1; p += 64 * kEvictAhead) {
        unsigned k[kEvictAhead];
#pragma unroll
        for (int i = 0; i < kEvictAhead; ++i) k[i] = keys[min(p + 64 * i + lane, hi - 1) - lo];
#pragma unroll
        for (int i = 0; i < kEvictAhead; ++i) {
            const int q = p + 64 * i + lane;
            const unsigned long long me = __ballot(q < w1 && k[i] == prefix);
            const bool take = q < w1 && (k[i] > prefix || (k[i] == prefix && eq + __popcll(me & below) < need));
            const unsigned long long mt = __ballot(take);
            if (take) kept[at + __popcll(mt & below)] = q;
            eq += __popcll(me);
            at += __popcll(mt);
        }
    }
}

// Rows of `bytes` bytes in pieces of T, N a thread and round (16 bytes; rows start anywhere, the last
// piece may overlap the one before it), pieces [u0, u1) of each; or the scores.
// The rows j0 .. budget - 1 of the kept list; target(j): L[j]; go(): whether
// anything moves, asked with the first loads in flight.
template <typename T, int N, typename Target, typename Go>
__device__ __forceinline__ void move_rows(const KvView& c, int seq, char* base, int64_t sp, int64_t ss, int bytes,
                                          int u0, int u1, const int32_t* kept, int j0, int budget, Target target, Go go) {
    // Lanes: the row's pieces, rounded up to a power of two, then rows
    typedef T U __attribute__((aligned(2)));
    const int un = u1 - u0, lg = un > 1 ? 32 - __builtin_clz(un - 1) : 0;
    const int u = threadIdx.x & ((1 << lg) - 1), rows = kEvictThreads >> lg, r0 = threadIdx.x >> lg;
    const int off = min((u0 + u) * (int)sizeof(T), bytes - (int)sizeof(T));
    const char* from[N];
    char* to[N];
    auto place = [&](int jr) {  // (budget < length <= 2^30)
#pragma unroll
        for (int x = 0; x < N; ++x) {
            const int j = jr + x * rows + r0;
            to[x] = nullptr;
            from[x] = base;  // (read and left, where nothing moves)
            if (j < budget && u < un) {
                const int dst = target(j), src = max(kept[j], 0);  // (-1: nothing moves)
                const int pf = kv_page(c, seq, src), pt = kv_page(c, seq, dst);
                if (src != dst && pf >= 0 && pt >= 0) {
                    from[x] = base + pf * sp + kv_slot(c, src) * ss + off;
                    to[x] = base + pt * sp + kv_slot(c, dst) * ss + off;
                }
            }
        }
    };
    place(j0);
    if (!go()) return;
    for (int jr = j0; jr < budget; jr += N * rows) {
        T val[N];
        char* dst[N];
#pragma unroll
        for (int x = 0; x < N; ++x) {
            dst[x] = to[x];
            val[x] = __builtin_nontemporal_load(reinterpret_cast<const U*>(from[x]));
        }
        place(jr + N * rows);  // (addresses: while the rows are on their way)
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // every load of the round is done
        __syncthreads();
#pragma unroll
        for (int x = 0; x < N; ++x)
            if (dst[x]) __builtin_nontemporal_store(val[x], reinterpret_cast<U*>(dst[x]));
    }
}

// What the selection says of a sequence that is cut: L[budget - 1] + 1 is its
// new length, so L[j] = j for every row where that is the budget.  (Fewer
// positions left than the budget: all stay where they are, and the list ends
// with -1.)
enum EvictMoves { kMoveNone, kMoveDense, kMoveHoles };
__device__ __forceinline__ EvictMoves evict_moves(const EvictArgs& a, int last_kept, int new_length) {
    if (last_kept < 0) return kMoveNone;
    return new_length == a.budget ? kMoveDense : kMoveHoles;
}

// blockIdx.y: key-value head; blockIdx.z: the parts of k's rows, of v's, the
// scores.
template <typename T>
__global__ __launch_bounds__(kEvictThreads, 8) void kv_evict_move_kernel(EvictArgs a, int es, int parts) {
    const KvView& c = a.c;
    __shared__ int list[kEvictThreads], counts[kEvictWaves];
    const int seq = blockIdx.x, h = blockIdx.y, z = blockIdx.z, n = kv_length(c, a.lengths[seq]);
    const int32_t* kept = a.kept + ((int64_t)seq * c.hkv + h) * a.budget;
    const int last = kept[a.budget - 1], len = a.new_lengths[seq];
    if (n <= a.budget) return;
    const int bytes = c.D * es, units = (bytes + (int)sizeof(T) - 1) / (int)sizeof(T), part = z % parts;
    char* base = static_cast<char*>(z < parts ? c.k : c.v) + c.sh * h * es;
    auto rows = [&](auto width, int j0, int j1, auto target, auto go) {
        constexpr int N = decltype(width)::value;
        if (z == 2 * parts)
            move_rows<float, N>(c, seq, reinterpret_cast<char*>(c.score + (int64_t)h * c.page),
                                (int64_t)c.hkv * c.page * 4, 4, 4, 0, 1, kept, j0, j1, target, go);
        else
            move_rows<T, N>(c, seq, base, c.sp * es, c.ss * es, bytes, units * part / parts,
                            units * (part + 1) / parts, kept, j0, j1, target, go);
    };
    rows(std::integral_constant<int, kMoveUnits>(), a.sink, a.budget, [](int j) { return j; },
         [&]() { return evict_moves(a, last, len) == kMoveDense; });
    if (evict_moves(a, last, len) != kMoveHoles) return;
    const int pages = kv_pages(c, n);
    for (int at = 0, j0 = 0; at < pages && j0 < a.budget; at += kEvictThreads) {
        const int j1 = j0 + live_entries<kEvictThreads>(c, seq, pages, at, list, counts) * c.page;
        // (a piece a thread: more would take registers that the other way needs)
        rows(std::integral_constant<int, 1>(), max(a.sink, j0), min(a.budget, j1), [&](int j) {
            const int e = kv_page_of(c, j - j0);
            return list[e] * c.page + j - j0 - e * c.page;
        }, []() { return true; });
        j0 = j1;
    }
}

// The same through a workspace, for calls of few heads and many rows: there the
// in-place rounds leave most of the chip idle, while here every row is copied
// on its own, all of them out (PUT false), then all of them in.  Staged:
// [seq][head][row][2 units pieces], and the scores.  Measured with 8 heads of
// 128 in bf16, both kernels against in place: 1200 rows 13 against 10 us, 2500
// 17 / 18, 5000 23 / 30, 30000 93 / 174.
template <bool PUT>
__global__ __launch_bounds__(256) void kv_evict_stage_kernel(EvictArgs a, int es) {
    typedef v4i U __attribute__((aligned(2)));
    const KvView& c = a.c;
    __shared__ int list[256], counts[4];
    const int seq = blockIdx.z, h = blockIdx.y, n = kv_length(c, a.lengths[seq]);
    const int64_t head = (int64_t)seq * c.hkv + h;
    const int32_t* kept = a.kept + head * a.budget;
    const int last = kept[a.budget - 1], len = a.new_lengths[seq];
    if (n <= a.budget) return;
    const EvictMoves moves = evict_moves(a, last, len);
    if (moves == kMoveNone) return;
    const int bytes = c.D * es, units = (bytes + 15) / 16, lg = 32 - __builtin_clz(2 * units - 1);
    const int u = threadIdx.x & ((1 << lg) - 1), rows = 256 >> lg;
    const int j0 = a.sink + blockIdx.x * kMoveUnits * rows + (threadIdx.x >> lg);
    int dst[kMoveUnits];  // L[j] of the thread's rows
#pragma unroll
    for (int i = 0; i < kMoveUnits; ++i) dst[i] = j0 + i * rows;
    if (moves == kMoveHoles) {
        const int pages = kv_pages(c, n), end = min(a.budget, a.sink + ((int)blockIdx.x + 1) * kMoveUnits * rows);
        for (int at = 0, before = 0; at < pages && before * c.page < end; at += 256) {
            const int m = live_entries<256>(c, seq, pages, at, list, counts);
#pragma unroll
            for (int i = 0; i < kMoveUnits; ++i) {
                const int j = j0 + i * rows - before * c.page, e = j < 0 ? -1 : kv_page_of(c, j);
                if (e >= 0 && e < m) dst[i] = list[e] * c.page + j - e * c.page;
            }
            before += m;
        }
    }
    if (u >= 2 * units) return;
    const bool val = u >= units;
    const int off = min((val ? u - units : u) * 16, bytes - 16);
    char* base = static_cast<char*>(val ? c.v : c.k) + c.sh * h * es + off;
    v4i* stage = a.stage + head * (a.budget - a.sink) * 2 * units + u;
    float* scores = a.stage_score + head * (a.budget - a.sink);
    v4i x[kMoveUnits];
    float sc[kMoveUnits];
    int64_t to[kMoveUnits];  // slot of the row that is written (PUT), -1: none
#pragma unroll
    for (int i = 0; i < kMoveUnits; ++i) {
        const int j = j0 + i * rows;
        to[i] = -1;
        if (j >= a.budget) continue;
        const int src = kept[j], pf = kv_page(c, seq, src), pt = kv_page(c, seq, dst[i]);
        if (src == dst[i] || pf < 0 || pt < 0) continue;
        to[i] = PUT ? pt : 0;
        if (PUT) {
            x[i] = stage[(int64_t)(j - a.sink) * 2 * units];
            if (u == 0) sc[i] = scores[j - a.sink];
        } else {
            const int slot = kv_slot(c, src);
            x[i] = __builtin_nontemporal_load(reinterpret_cast<const U*>(base + (pf * c.sp + slot * c.ss) * es));
            if (u == 0) sc[i] = c.score[((int64_t)pf * c.hkv + h) * c.page + slot];
        }
    }
#pragma unroll
    for (int i = 0; i < kMoveUnits; ++i) {
        const int j = j0 + i * rows;
        if (to[i] < 0) continue;
        if (PUT) {
            const int slot = kv_slot(c, dst[i]);
            *reinterpret_cast<U*>(base + (to[i] * c.sp + slot * c.ss) * es) = x[i];
            if (u == 0) c.score[(to[i] * c.hkv + h) * c.page + slot] = sc[i];
        } else {
            stage[(int64_t)(j - a.sink) * 2 * units] = x[i];
            if (u == 0) scores[j - a.sink] = sc[i];
        }
    }
}

size_t evict_key_bytes(const EvictArgs& a) {
    const int64_t mid = (int64_t)a.c.max_pages * a.c.page - a.sink - a.recent;
    return mid > kEvictRegs * kEvictThreads ? (size_t)(a.c.hkv * mid) * sizeof(unsigned) : 0;
}

namespace {

struct EvictPlan {
    size_t keys, stage, scores;  // bytes of the workspace's parts
    int parts;                   // of a row, moved in place
    bool moves, staged;
};

EvictPlan make_plan(int dtype, const EvictArgs& a, int cus) {
    EvictPlan pl;
    const int64_t cap = (int64_t)a.c.max_pages * a.c.page;
    const int64_t heads = (int64_t)a.c.nseq * a.c.hkv, kept = a.budget - a.sink;
    pl.keys = ((size_t)a.c.nseq * evict_key_bytes(a) + 255) / 256 * 256;
    pl.moves = kept > 0 && cap > a.budget;
    // Parts of a row until two workgroups per compute unit, of four pieces at least
    const int bytes = a.c.D * (dtype == XT_F32 ? 4 : 2), units = (bytes + 15) / 16;
    pl.parts = bytes < 16 ? 1 : (int)std::max<int64_t>(1, std::min<int64_t>(units / 4, (int64_t)cus / heads));
    // Through the workspace where that leaves half the compute units without a
    // workgroup and there are rows enough to pay for the second kernel.  Whole
    // calls, staged against in place, 6000 / 12000 rows: 12 heads of 128 in bf16 (96
    // workgroups) 96 / 165 us against 104 / 190, 16 heads (128) 104 / 181 against
    // 101 / 185, 24 heads (192) 124 / 217 against 110 / 200, 32 heads (256) 138 / 270
    // against 117 / 220; 8 heads in f32 (128) 103 / 178 against 102 / 189, 16 heads
    // (256) 136 / 266 against 121 / 225.  4096 rows of 8 heads: 68 either way; of one
    // head of 64 in f16 52 against 67, and 33 against 37 at 2000 (not taken).
    const double stage = (double)heads * kept * (32.0 * units + 4);
    pl.staged = pl.moves && bytes >= 16 && 4 * heads * pl.parts <= cus && kept >= 4096 && stage < 4e9;
    pl.stage = pl.staged ? (size_t)(heads * kept) * 32 * units : 0;
    pl.scores = pl.staged ? (size_t)(heads * kept) * sizeof(float) : 0;
    return pl;
}

}  // namespace

size_t evict_workspace(int dtype, const EvictArgs& a, int cus) {
    const EvictPlan pl = make_plan(dtype, a, cus);
    return pl.keys + pl.stage + pl.scores;
}

hipError_t launch_kv_evict(int dtype, EvictArgs a, int cus, void* ws, hipStream_t s) {
    const EvictPlan pl = make_plan(dtype, a, cus);
    const KvView& c = a.c;
    a.keys = static_cast<unsigned*>(ws);
    a.ldk = (int64_t)c.max_pages * c.page - a.sink - a.recent;
    a.stage = reinterpret_cast<v4i*>(static_cast<char*>(ws) + pl.keys);
    a.stage_score = reinterpret_cast<float*>(static_cast<char*>(ws) + pl.keys + pl.stage);
    const int es = dtype == XT_F32 ? 4 : 2, units = (c.D * es + 15) / 16;
    hipError_t e;
    if (pl.keys) {
        const int64_t tiles = std::min<int64_t>((a.ldk + kEvictTile - 1) / kEvictTile, 65535);
        kv_evict_keys_kernel<<<dim3((unsigned)c.nseq, (unsigned)c.hkv, (unsigned)tiles), 256, 0, s>>>(a);
        if ((e = hipGetLastError()) != hipSuccess) return e;
    }
    kv_evict_select_kernel<<<dim3((unsigned)c.nseq, (unsigned)c.hkv), kEvictThreads, 0, s>>>(a);
    if ((e = hipGetLastError()) != hipSuccess || !pl.moves) return e;
    if (pl.staged) {
        int lg = 0;
        while ((1 << lg) < 2 * units) ++lg;
        const int rows = kMoveUnits * (256 >> lg);  // of a workgroup
        const dim3 grid((unsigned)((a.budget - a.sink + rows - 1) / rows), (unsigned)c.hkv, (unsigned)c.nseq);
        kv_evict_stage_kernel<false><<<grid, 256, 0, s>>>(a, es);
        if ((e = hipGetLastError()) != hipSuccess) return e;
        kv_evict_stage_kernel<true><<<grid, 256, 0, s>>>(a, es);
        return hipGetLastError();
    }
    const dim3 grid((unsigned)c.nseq, (unsigned)c.hkv, (unsigned)(2 * pl.parts + 1));
    if (c.D * es >= 16)
        kv_evict_move_kernel<v4i><<<grid, kEvictThreads, 0, s>>>(a, es, pl.parts);
    else
        kv_evict_move_kernel<short><<<grid, kEvictThreads, 0, s>>>(a, es, pl.parts);
    return hipGetLastError();
}

}  // namespace xt
