// Token probabilities of rows of logits: ln p of given tokens, entropy, the
// most likely tokens.
//
// m = max x, z = sum over all but one maximum of exp(x - m),
// ln p(t) = x_t - m - ln(1 + z), H = ln(1 + z) - sum (x - m) exp(x - m) / (1 + z).
// Leaving the maximum's own 1 out of the sum keeps ln p of an almost certain
// token exact to its last bits.  Logits of -inf have p = 0; a row of nothing
// else gives ln p = -inf and H = 0.
//
// The logits are read once: HBM bounds large calls, the chain of load,
// reduction and selection small ones.  A workgroup walks its slice of a row in
// tiles of 8192 logits that stay in registers from the maximum over the sums to
// the selection, the next tile in flight meanwhile; sums are per thread,
// relative to the workgroup's running maximum, and reduced once at the end.  A
// row is cut into slices only as far as there are too few rows for the chip;
// the workgroup that ends a row's last slice joins them (results and count at
// device scope, as the chip's eight L2s need it).
//
// Selection of the `top` largest: a wave's q-th largest lane maximum, q = top /
// 8, is reached by at least q of its logits, so the minimum of that over the
// eight waves is by `top` of the tile's, and by hardly more than twice as many.
// Those go to LDS, each counts how many are before it, and the first `top` in
// that order are the list that the next tile's candidates have to beat.  Where
// that fails (ties beyond the buffer, fewer finite logits than `top`) the tile
// is selected from by the digits of its logits.
//
// Measured: 1024 rows of 128256 f32 logits 84 us without alternatives (6.3
// TB/s), 91 / 124 / 176 with 1 / 20 / 64; of f16 or bf16 65 us (4.0 TB/s) and 107 / 157 with
// 20 / 64, where the instructions count: the exponentials, and for alternatives
// the barriers of each tile.  One row of f32 with 20 10.7 us, where the chain of
// load, reduction, selection and join counts.
#include <algorithm>

#include "xtern_cache.h"

namespace xt {

typedef unsigned long long u64;

constexpr int kProbsThreads = 512;
constexpr int kProbsWaves = kProbsThreads / 64;
constexpr int kProbsPer = 16;                              // logits of a thread and tile
constexpr int kProbsTile = kProbsThreads * kProbsPer;
constexpr int kProbsTop = 64;
constexpr int kProbsCand = 1024;                           // candidates of a tile, with the list before it
constexpr int kProbsSlices = 64;

// Slices of a row: slice s is tiles [s * per, (s + 1) * per).
struct ProbsPlan {
    int slices, per, tiles;
    u64* stats;       // [M][slices][2]: m and z, xz and the count of the maximum
    u64* keys;        // [M][slices][top]
    unsigned* count;  // [M]: slices done, zero between calls
};

// The first `top` of keys[0 .. n) in descending order, to list[0 .. min(top,
// n)): each counts how many are larger, four threads a key.  Zeros follow the
// keys up to a multiple of 32.
__device__ __forceinline__ void probs_rank(const u64* keys, int n, int top, u64* list) {
    const int part = threadIdx.x & 3;
    for (int i = threadIdx.x >> 2; i < n; i += kProbsThreads / 4) {
        const u64 k = keys[i];
        int before = 0;
        for (int j = part; j < n; j += 32) {
            u64 o[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) o[u] = keys[j + 4 * u];
#pragma unroll
            for (int u = 0; u < 8; ++u) before += o[u] > k;
        }
        before += __builtin_amdgcn_mov_dpp(before, 0xb1, 0xf, 0xf, true);  // (the four lanes of a quad)
        before += __builtin_amdgcn_mov_dpp(before, 0x4e, 0xf, 0xf, true);
        if (part == 0 && before < top) list[before] = k;
    }
}

// Order of the alternatives: larger value first, then the lower index; NaN
// behind everything, no element (0) behind that.
__device__ __forceinline__ u64 probs_key(float x, int i) {
    const float f = x + 0.0f;  // (-0 counts as +0)
    unsigned u = __float_as_uint(f);
    u = f != f ? 0u : u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u);
    return ((u64)u << 32) | (unsigned)~i;
}
__device__ __forceinline__ float key_value(u64 k) {
    const unsigned u = (unsigned)(k >> 32);
    return __uint_as_float((u >> 31) ? u ^ 0x80000000u : ~u);
}
__device__ __forceinline__ int key_index(u64 k) { return (int)~(unsigned)k; }

// Reductions over the wave, the result in every lane: within 16 lanes by DPP
// (quads, halves of a row, rows: each step meets lanes that hold the same
// value already), then by lane swaps.
template <typename Op>
__device__ __forceinline__ float wave_all(float v, Op op) {
    v = op(v, __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0xb1, 0xf, 0xf, true)));   // quad_perm 1,0,3,2
    v = op(v, __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0x4e, 0xf, 0xf, true)));   // quad_perm 2,3,0,1
    v = op(v, __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0x141, 0xf, 0xf, true)));  // row_half_mirror
    v = op(v, __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0x140, 0xf, 0xf, true)));  // row_mirror
    auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = op(__uint_as_float(a[0]), __uint_as_float(a[1]));
    auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return op(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float wave_max_f(float v) {
    return wave_all(v, [](float p, float q) { return fmaxf(p, q); });
}
__device__ __forceinline__ float wave_sum_f(float v) {
    return wave_all(v, [](float p, float q) { return p + q; });
}

// Sums relative to m, of which `c` logits are m itself; to a larger maximum.
struct ProbsSum {
    float m, z, xz, c;
    __device__ __forceinline__ void raise(float to) {
        if (!(to > m)) return;
        if (m == -INFINITY) {
            z = z == z ? 0.0f : z;  // (a NaN stays)
            xz = 0.0f;
        } else {
            const float d = m - to, f = __builtin_amdgcn_exp2f(d * 1.44269504f), s = z + c;
            xz = f == 0.0f ? 0.0f : (xz + d * s) * f;
            z = z == z ? (f == 0.0f ? 0.0f : s * f) : z;
        }
        m = to;
        c = 0.0f;
    }
};

__device__ __forceinline__ void st_device(u64* p, u64 v) {
    __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ u64 ld_device(const u64* p) {
    return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ u64 pack2(float lo, float hi) {
    return ((u64)__float_as_uint(hi) << 32) | __float_as_uint(lo);
}
__device__ __forceinline__ float low(u64 v) { return __uint_as_float((unsigned)v); }
__device__ __forceinline__ float high(u64 v) { return __uint_as_float((unsigned)(v >> 32)); }

struct ProbsLds {
    float wmax[2][kProbsWaves], wbound[2][kProbsWaves];
    float sums[3][kProbsWaves];
    u64 cand[kProbsCand];
    u64 list[kProbsTop];
    u64 wbest[kProbsWaves + 1];
    int count, last;
};

// The row's results from its sums and its list of the `top` first keys.
template <int DT>
__device__ void probs_finish(const ProbsArgs& a, int64_t r, ProbsSum s, const u64* list) {
    typedef Elem<DT> E;
    const typename E::T* x = static_cast<const typename E::T*>(a.x) + r * a.ld;
    s.z += s.c - 1.0f;  // one maximum left out
    const bool none = s.m == -INFINITY && s.z == s.z;
    const float ln = s.m == INFINITY ? NAN : log1pf(s.z);
    if (threadIdx.x == 0) a.entropy[r] = none ? 0.0f : ln - s.xz / (1.0f + s.z);
    auto lnp = [&](float v) { return none ? v : v - s.m - ln; };
    for (int i = threadIdx.x; i < a.T; i += kProbsThreads) {
        const int tok = a.tokens[r * a.T + i];
        a.lp[r * a.T + i] = tok < 0 ? 0.0f : (tok < a.V ? lnp(E::get(x[tok])) : NAN);
    }
    for (int i = threadIdx.x; i < a.top; i += kProbsThreads) {
        a.ids[r * a.top + i] = key_index(list[i]);
        a.top_lp[r * a.top + i] = lnp(key_value(list[i]));
    }
}

// The first `top` of a tile's logits and of the list before it, whatever they
// are: the last one's value by four passes of a histogram, then everything
// above it, and of its equals the list's and then the lowest indices.
template <int W, typename Index>
__device__ void probs_select(const float* x, Index index, int V, int valid, int top, int* have, ProbsLds& lds) {
    const int t = threadIdx.x, wave = t >> 6, lane = t & 63;
    const u64 mine = t < *have ? lds.list[t] : 0;  // (wave 0: an entry a lane)
    const unsigned mine_v = (unsigned)(mine >> 32);
    int* hist = reinterpret_cast<int*>(lds.cand);  // [4][256]
    __syncthreads();
    for (int i = t; i < 4 * 256; i += kProbsThreads) hist[i] = 0;
    __syncthreads();
    const int want = min(top, *have + valid);
    int need = want;
    unsigned value = 0;
    auto word = [&](int i) { return (unsigned)(probs_key(x[i], 0) >> 32); };
    for (int pass = 0; pass < 4; ++pass) {
        const int shift = 24 - 8 * pass;
        const unsigned mask = pass ? ~0u << (shift + 8) : 0u;
#pragma unroll
        for (int i = 0; i < kProbsPer; ++i)
            hist_add(hist + 256 * pass, (word(i) >> shift) & 255, index(i) < V && (word(i) & mask) == value);
        if (mine && (mine_v & mask) == value) atomicAdd(&hist[256 * pass + ((mine_v >> shift) & 255)], 1);
        __syncthreads();
        int left;
        value |= (unsigned)radix_bin(hist + 256 * pass, need, &left) << shift;
        need = left;
    }
    __syncthreads();
    // `need` of the equals: the list's entries come first
    const u64 of_list = __ballot(mine && mine_v == value);
    if (t == 0) lds.wbest[kProbsWaves] = of_list;
    // The tile's equals before this thread's, for each run of W indices: 16
    // bits each, 8192 in all at most
    u64 eq = 0;
#pragma unroll
    for (int i = 0; i < kProbsPer; ++i)
        if (index(i) < V && word(i) == value) eq += (u64)1 << (16 * (i / W));
    u64 before = eq;
    for (int o = 1; o < 64; o <<= 1) {
        const u64 y = __shfl_up(before, o);
        if (lane >= o) before += y;
    }
    if (lane == 63) lds.wbest[wave] = before;
    before -= eq;
    for (int i = t; i < 96; i += kProbsThreads) lds.cand[i] = 0;
    if (t == 0) lds.count = 0;
    __syncthreads();
    const u64 listed = lds.wbest[kProbsWaves];
    u64 total = 0;
    for (int w = 0; w < kProbsWaves; ++w) {
        if (w < wave) before += lds.wbest[w];
        total += lds.wbest[w];
    }
    const int rest = need - min(need, (int)__popcll(listed));
    if (mine && (mine_v > value || (mine_v == value && (int)__popcll(listed & (((u64)1 << lane) - 1)) < need)))
        lds.cand[atomicAdd(&lds.count, 1)] = mine;
    int run = 0;  // the tile's equals before run i / W
#pragma unroll
    for (int i = 0; i < kProbsPer; ++i) {
        if (i && i % W == 0) run += (int)((total >> (16 * (i / W - 1))) & 0xffff);
        if (index(i) >= V) continue;
        bool take = word(i) > value;
        if (word(i) == value) {
            take = run + (int)((before >> (16 * (i / W))) & 0xffff) < rest;
            before += (u64)1 << (16 * (i / W));
        }
        if (take) lds.cand[atomicAdd(&lds.count, 1)] = probs_key(x[i], index(i));
    }
    __syncthreads();
    probs_rank(lds.cand, want, top, lds.list);
    __syncthreads();
    *have = want;
}

// 16 logits of a thread: vectors of 16 bytes (W logits), vector v at
// tile + (v * threads + thread) * W.
template <int DT>
struct ProbsTileRegs {
    static constexpr int W = DT == XT_F32 ? 4 : 8, NV = kProbsPer / W;
    typedef typename Elem<DT>::T T;
    typedef T Vec __attribute__((ext_vector_type(W)));
    typedef Vec VecU __attribute__((aligned(sizeof(T))));
    Vec v[NV];
    __device__ __forceinline__ void load(const T* x, int64_t base, int V) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int64_t at = base + (int64_t)(i * kProbsThreads + (int)threadIdx.x) * W;
            if (at + W <= V) {
                v[i] = __builtin_nontemporal_load(reinterpret_cast<const VecU*>(x + at));
            } else {
#pragma unroll
                for (int j = 0; j < W; ++j) v[i][j] = at + j < V ? x[at + j] : (T)-INFINITY;
            }
        }
    }
};

// Joins a row's slices: the sums, and of the lists (each in descending order)
// the first `top`.  With q = ceil(top / slices), the slices' q-th entries have
// a minimum that at least `top` entries reach: only those are ranked.
template <int DT>
__device__ void probs_join(const ProbsArgs& a, const ProbsPlan& pl, int64_t r, u64* keys, ProbsLds& lds) {
    const int n = pl.slices * a.top, sl = min((int)(threadIdx.x & 63), pl.slices - 1);
    constexpr int kMine = kProbsSlices * kProbsTop / kProbsThreads;
    u64 mine[kMine];
#pragma unroll
    for (int i = 0; i < kMine; ++i) {
        const int at = i * kProbsThreads + threadIdx.x;
        mine[i] = at < n ? ld_device(pl.keys + r * n + at) : 0;
    }
    const u64 s0 = ld_device(pl.stats + (r * pl.slices + sl) * 2), s1 = ld_device(pl.stats + (r * pl.slices + sl) * 2 + 1);
    u64 bound = 0;
    if (a.top) {
        bound = ld_device(pl.keys + r * n + (int64_t)sl * a.top + (a.top + pl.slices - 1) / pl.slices - 1);
        for (int o = 32; o; o >>= 1) bound = min(bound, __shfl_xor(bound, o));
    }
    ProbsSum s{low(s0), high(s0), low(s1), high(s1)};
    s.raise(wave_max_f(s.m));
    const bool in = (int)(threadIdx.x & 63) < pl.slices;
    s.z = wave_sum_f(in ? s.z : 0.0f);
    s.xz = wave_sum_f(in ? s.xz : 0.0f);
    s.c = wave_sum_f(in ? s.c : 0.0f);
    for (int i = threadIdx.x; i < (n + 31) / 32 * 32; i += kProbsThreads) keys[i] = 0;
    if (threadIdx.x == 0) lds.count = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kMine; ++i)
        if (mine[i] && mine[i] >= bound) keys[atomicAdd(&lds.count, 1)] = mine[i];
    __syncthreads();
    probs_rank(keys, lds.count, a.top, lds.list);
    __syncthreads();
    probs_finish<DT>(a, r, s, lds.list);
}

template <int DT>
__global__ __launch_bounds__(kProbsThreads, 4) void token_logprobs_kernel(ProbsArgs a, ProbsPlan pl) {
    typedef ProbsTileRegs<DT> R;
    typedef typename R::T T;
    __shared__ ProbsLds lds;
    __shared__ u64 join_keys[kProbsSlices * kProbsTop];
    const int t = threadIdx.x, wave = t >> 6, lane = t & 63;
    const int64_t r = blockIdx.x / pl.slices;
    const int slice = blockIdx.x % pl.slices;
    const T* row = static_cast<const T*>(a.x) + r * a.ld;
    const int t0 = slice * pl.per, t1 = min(t0 + pl.per, pl.tiles);
    int have = 0, dirty = kProbsCand;  // entries of the list; of the buffer, to be cleared
    const int quota = (a.top + kProbsWaves - 1) / kProbsWaves;
    ProbsSum s{-INFINITY, 0.0f, 0.0f, 0.0f};
    R next;
    next.load(row, (int64_t)t0 * kProbsTile, a.V);
    for (int tile = t0; tile < t1; ++tile) {
        const int base = tile * kProbsTile;  // (V <= 2^30)
        float x[kProbsPer];
#pragma unroll
        for (int i = 0; i < kProbsPer; ++i) x[i] = Elem<DT>::get(next.v[i / R::W][i % R::W]);
        if (tile + 1 < t1) next.load(row, (int64_t)(tile + 1) * kProbsTile, a.V);
        float mx = -INFINITY;
#pragma unroll
        for (int i = 0; i < kProbsPer; ++i) mx = fmaxf(mx, x[i]);
        // the wave's `quota`-th largest of its lanes' maxima
        const float wm = wave_max_f(mx);
        float wb = wm, rest = mx;
        // (a full list's last; a wave without anything above it has no say in
        // the bound, and then there is none)
        const bool full = have == a.top;
        const float last = full && a.top ? key_value(lds.list[a.top - 1]) : -INFINITY;
        if (full && !(wm > last)) {
            wb = -INFINITY;
        } else {
            for (int i = 1; i < quota; ++i) {
                const u64 holds = __ballot(rest == wb);
                if (holds && lane == __builtin_ctzll(holds)) rest = -INFINITY;
                wb = wave_max_f(rest);
            }
        }
        if (lane == 0) {
            lds.wmax[tile & 1][wave] = wm;
            lds.wbound[tile & 1][wave] = wb;
        }
        for (int i = t; i < dirty; i += kProbsThreads) lds.cand[i] = 0;
        dirty = 0;
        if (t == 0) lds.count = have;
        __syncthreads();
        float m = lds.wmax[tile & 1][0], bound = lds.wbound[tile & 1][0];
#pragma unroll
        for (int w = 1; w < kProbsWaves; ++w) {
            m = fmaxf(m, lds.wmax[tile & 1][w]);
            bound = fminf(bound, lds.wbound[tile & 1][w]);
        }
        const float tile_max = m;
        m = fmaxf(m, s.m);
        s.raise(m);
        if (mx == m) {
            // this thread holds a maximum (or nothing): summed apart from the rest
            float z = 0.0f;
#pragma unroll
            for (int i = 0; i < kProbsPer; ++i) {
                const float d = x[i] - m, e = __builtin_amdgcn_exp2f(d * 1.44269504f);
                if (x[i] == m) {
                    s.c += 1.0f;
                } else {
                    z += e;
                    s.xz = fmaf(fmaxf(d, -200.0f), e, s.xz);
                }
            }
            s.z += z;
        } else {
            float z = 0.0f;
#pragma unroll
            for (int i = 0; i < kProbsPer; ++i) {
                const float d = x[i] - m, e = __builtin_amdgcn_exp2f(d * 1.44269504f);
                z += e;
                s.xz = fmaf(fmaxf(d, -200.0f), e, s.xz);  // (e is 0 there; -inf would give NaN)
            }
            s.z += z;
        }
        if (!a.top) continue;
        const int valid = min(kProbsTile, a.V - base);
        // (uniform: nothing of the tile comes before the list's last)
        if (full && !(tile_max > last)) {
            if (last == last) continue;
        }
        if (t < have) lds.cand[t] = lds.list[t];
        const int at = base + t * R::W;  // of x[0]
        auto index = [&](int i) { return at + (i / R::W) * kProbsThreads * R::W + i % R::W; };
        if (mx >= bound && mx > last) {
            int hits = 0;
#pragma unroll
            for (int i = 0; i < kProbsPer; ++i) hits += x[i] >= bound && x[i] > last;
            int pos = atomicAdd(&lds.count, hits);
#pragma unroll
            for (int i = 0; i < kProbsPer; ++i)
                if (x[i] >= bound && x[i] > last) {
                    if (pos < kProbsCand) lds.cand[pos] = probs_key(x[i], index(i));
                    ++pos;
                }
        }
        __syncthreads();
        const int n = lds.count;
        dirty = min(n, kProbsCand);
        if (n > kProbsCand || n < min(a.top, have + valid) || (full && last != last)) {
            probs_select<R::W>(x, index, a.V, valid, a.top, &have, lds);
            dirty = kProbsCand;
            continue;
        }
        probs_rank(lds.cand, n, a.top, lds.list);
        have = min(a.top, n);
        __syncthreads();
    }
    // the workgroup's sums
    s.z = wave_sum_f(s.z);
    s.xz = wave_sum_f(s.xz);
    s.c = wave_sum_f(s.c);
    __syncthreads();
    if (lane == 0) {
        lds.sums[0][wave] = s.z;
        lds.sums[1][wave] = s.xz;
        lds.sums[2][wave] = s.c;
    }
    __syncthreads();
    s.z = s.xz = s.c = 0.0f;
    for (int w = 0; w < kProbsWaves; ++w) {
        s.z += lds.sums[0][w];
        s.xz += lds.sums[1][w];
        s.c += lds.sums[2][w];
    }
    if (pl.slices == 1) {
        probs_finish<DT>(a, r, s, lds.list);
        return;
    }
    if (t == 0) {
        st_device(pl.stats + (int64_t)blockIdx.x * 2, pack2(s.m, s.z));
        st_device(pl.stats + (int64_t)blockIdx.x * 2 + 1, pack2(s.xz, s.c));
    }
    for (int i = t; i < a.top; i += kProbsThreads)
        st_device(pl.keys + (int64_t)blockIdx.x * a.top + i, i < have ? lds.list[i] : 0);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // every store has arrived
    __syncthreads();
    // (the count wraps to zero by itself, for the next call)
    if (t == 0) lds.last = atomicInc(pl.count + r, (unsigned)pl.slices - 1) == (unsigned)pl.slices - 1;
    __syncthreads();
    if (lds.last) probs_join<DT>(a, pl, r, join_keys, lds);
}

namespace {

ProbsPlan make_plan(const ProbsArgs& a, int cus) {
    ProbsPlan pl;
    pl.tiles = (a.V + kProbsTile - 1) / kProbsTile;
    // slices until two workgroups per compute unit (what it holds, by registers).
    // One of 128256 f32 logits each, 20 alternatives, against slices for four and
    // for eight a unit: 37 rows 18 us (21, 20), 128 rows 27 (37, 47), 512 rows 63
    // (74, 90); 300 rows 59 (55, 68).  From 513 rows on, 85 us, a row is one slice,
    // and the ones that do not fit at once wait for the others.
    const int64_t want = std::max<int64_t>(1, 2 * (int64_t)cus / std::max<int64_t>(a.M, 1));
    const int slices = (int)std::min<int64_t>(std::min<int64_t>(want, kProbsSlices), pl.tiles);
    pl.per = (pl.tiles + slices - 1) / slices;
    pl.slices = (pl.tiles + pl.per - 1) / pl.per;
    pl.stats = pl.keys = nullptr;
    pl.count = nullptr;
    return pl;
}

template <int DT>
hipError_t launch(const ProbsArgs& a, const ProbsPlan& pl, hipStream_t s) {
    token_logprobs_kernel<DT><<<(unsigned)(a.M * pl.slices), kProbsThreads, 0, s>>>(a, pl);
    return hipGetLastError();
}

}  // namespace

size_t token_logprobs_workspace(const ProbsArgs& a, int cus, size_t* counters) {
    const ProbsPlan pl = make_plan(a, cus);
    *counters = pl.slices == 1 ? 0 : (size_t)a.M * sizeof(unsigned);
    return pl.slices == 1 ? 0 : (size_t)a.M * pl.slices * (2 + (size_t)a.top) * sizeof(u64);
}

hipError_t launch_token_logprobs(int dtype, const ProbsArgs& a, int cus, void* ws, void* counters, hipStream_t s) {
    ProbsPlan pl = make_plan(a, cus);
    pl.stats = static_cast<u64*>(ws);
    pl.keys = pl.stats + (size_t)a.M * pl.slices * 2;
    pl.count = static_cast<unsigned*>(counters);
    switch (dtype) {
        case XT_F32: return launch<XT_F32>(a, pl, s);
        case XT_F16: return launch<XT_F16>(a, pl, s);
        default: return launch<XT_BF16>(a, pl, s);
    }
}

}  // namespace xt
