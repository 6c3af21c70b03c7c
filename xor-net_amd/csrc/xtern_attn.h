// What the attention kernels of the 16- and 32-bit caches (xtern_attn.hip) and
// of the 8-bit ones (xtern_attn8.hip) share: what a row sees of its sequence,
// the split of all rows' positions over the workgroups, and the join of the
// parts.
#pragma once
#include <algorithm>

#include "xtern_cache.h"

namespace xt {

typedef float v4f __attribute__((ext_vector_type(4)));
typedef int v2i __attribute__((ext_vector_type(2)));
// (rows may start at any element: the hardware loads unaligned vectors)
typedef v4f v4fu __attribute__((aligned(4)));

constexpr int kAttnThreads = 256;
constexpr int kAttnWaves = kAttnThreads / 64;
constexpr int kAttnStep = 128;       // positions: the unit of the split
constexpr int kAttnPlanRows = 1024;  // rows whose work is split by its total

// Asks for all lines of a kernel's arguments, ARGS one after the other, at once:
// each is a trip to memory for the workgroup that reads it first, and the code
// takes them one by one as it needs them.  (700 positions of 20 and 5 heads: 11.2
// us of kernel, 11.35 without; 131072 positions 95.4 and 95.9.)
template <typename... ARGS>
__device__ __forceinline__ void attn_touch_args() {
    typedef const __attribute__((address_space(4))) int* Kernarg;
    const Kernarg k = (Kernarg)__builtin_amdgcn_kernarg_segment_ptr();
    constexpr int kLines = ((int)(sizeof(ARGS) + ...) + 63) / 64;
    static_assert(kLines <= 6);
    int x[6];
#pragma unroll
    for (int i = 0; i < 6; ++i) x[i] = k[16 * (i < kLines ? i : 0)];
    asm volatile("" ::"s"(x[0]), "s"(x[1]), "s"(x[2]), "s"(x[3]), "s"(x[4]), "s"(x[5]));
}

// What is attended with one pass over the cache: a unit, one row or (8-bit
// caches) up to `unit_rows` of the `tokens` rows of one sequence.
struct AttnUnit {
    int row, rows;  // [row, row + rows)
    int seq;
};
__device__ __forceinline__ AttnUnit attn_unit(const AttnArgs& a, int u) {
    AttnUnit x;
    if (a.tokens == 1) {
        x.row = u;
        x.rows = 1;
        x.seq = a.seq ? a.seq[u] : u;
        return x;
    }
    // (row0 > 0: units are rows, these the ones from row0 on)
    const int v = u + a.row0, group = fast_quot(v, a.by_units), first = (v - group * a.units) * a.unit_rows;
    x.row = group * a.tokens + first - a.row0;
    x.rows = min(a.unit_rows, a.tokens - first);
    x.seq = a.seq ? a.seq[group * a.tokens] : group;
    return x;
}

// The positions that some row of a unit sees, side by side: position i of them
// is position i of the sequence below `sink`, i + gap from there on.
struct AttnSpan {
    int n, gap;
    int seq;  // (the unit's)
};
// SPANS false: units are rows and see all of their sequences' positions.
template <bool SPANS>
__device__ __forceinline__ AttnSpan attn_span(const AttnArgs& a, int u) {
    if constexpr (!SPANS) {
        const int seq = a.seq ? a.seq[u] : u;
        return AttnSpan{(unsigned)seq < (unsigned)a.c.nseq ? kv_length(a.c, a.lengths[u]) : 0, 0, seq};
    }
    const AttnUnit x = attn_unit(a, u);
    AttnSpan s{0, 0, x.seq};
    int least = a.c.max_pages * a.c.page;  // (at most 2^30)
    if (x.rows == 1) {
        s.n = kv_length(a.c, a.lengths[x.row]);
    } else {
        for (int t = 0; t < x.rows; t += 4) {  // (four loads in flight)
            int n[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) n[i] = a.lengths[x.row + min(t + i, x.rows - 1)];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                n[i] = kv_length(a.c, n[i]);
                s.n = max(s.n, n[i]);
                if (n[i] > 0) least = min(least, n[i]);
            }
        }
    }
    if ((unsigned)x.seq >= (unsigned)a.c.nseq) return AttnSpan{0, 0, x.seq};
    s.gap = max(0, min(s.n, least) - a.window - a.sink);
    s.n -= s.gap;
    return s;
}
template <bool SPANS>
__device__ __forceinline__ int attn_pos(const AttnArgs& a, int gap, int i) {
    return SPANS ? i + (i >= a.sink ? gap : 0) : i;
}

// The split.  The steps of all rows (an empty row has one, for its zeros) form
// one line, cut into equal shares for as many workgroups as run at once: rows
// of any lengths keep all of them busy to the end.  A share may cover the end
// of one row, whole rows and the start of another: its segments.  A segment's
// sums go to slot (workgroup + row), which both grow along the line, so no two
// segments share one and a row's slots are consecutive.
// More than kAttnPlanRows rows: one workgroup per row and group of heads.  With
// that many rows of like lengths they fill the chip by themselves, and the
// line costs its scan: 1000 / 2000 rows of up to 2000 positions, 32 and 8 heads
// of 128 in bf16, 699 / 1415 us on the line, 658 / 1331 a workgroup each; of 2000 to
// 4000, 1000 rows, 1927 against 2040.  What the limit costs is a long row among
// many short ones: 1000 rows, one of 60000 positions and the others of 100, 193
// us on the line and 1018 without; 1100 rows 972 as it is, 210 on the line.
// Parts (8-bit caches, whose cost per position is half of the others'): with half
// as many units as workgroups at most, each unit is cut by itself, into as many
// equal parts as the shortest length allows that gives every part a workgroup of
// its own.  A share then is one segment; on the line most shares have the end of
// one unit and the start of the next, and a segment costs as much as 400
// positions.  24 sequences of 5 tokens and 1032 positions, 20 and 5 heads of 128: 34
// us on the line, 26 in parts; 40 of one token and 1028 30 and 24; 30 of 4000, 32 and
// 8 heads, 53 and 51; 50 of 3000, which are more than half the workgroups, 61.6 (on
// the line, as it is) and 61.8.
// The workgroup that ends the last of a row's segments joins them, from 32
// segments on in two levels (groups of 32, then the groups): what one
// workgroup can read at device scope, about 20 GB/s, bounds a join.  Segments
// and counts are written and read at device scope, as the chip's eight L2s
// need it (a fence would write back and drop whole caches).
struct AttnPlan {
    float* part_o;   // [slots][hy][16][dp], unnormalised, relative to the segment's maximum
    float* part_ml;  // [slots][hy][16][2]: maximum (base 2), sum
    unsigned* count; // [slots][hy]: segments of the group done that begins there; zero between calls
    unsigned* tops;  // [R][hy]: groups of the row done; zero between calls
    float* ml;       // accumulate: maximum and sum of the whole row, [R][hq][2]
    int dp;          // D, made even
    float* s;        // accumulate: S in base 2, [R][hq][cap]
    int64_t cap;     // positions that a row may see, its part of s: a multiple of 32
    int hy;          // workgroups per share: kv heads x tiles of 16 query heads
    int tiles;       // of 16 query heads per kv head
    int shares;      // at most
    double inv_shares;
    int units;       // of the call
    bool parts;      // a share is a part of one unit (8-bit caches)
    bool per_row;
};

// A unit's part of the line, and of it what one share covers.
struct AttnSeg {
    int row, n, gap;  // the unit, its positions
    int seq;          // its sequence
    int p0, p1;       // the share's [p0, p1) of them
    int nc;           // segments of the unit
    int64_t slot;     // of its first one
};

__device__ __forceinline__ int attn_steps(int len) { return max(1, (len + kAttnStep - 1) / kAttnStep); }

// The line as every wave of the workgroup sees it: 64 units, a lane each, in
// registers (no barrier), or the units' ends in LDS.  PARTS: the plan may ask for
// parts.
template <bool SPANS, bool PARTS>
struct AttnLine {
    const AttnArgs& a;
    const AttnPlan& pl;
    int len, gap, seq, upto;  // the lane's unit (at most 64)
    int64_t* ends;       // LDS, [units] (more)
    int R;               // units
    int64_t total;       // steps
    int64_t per;         // steps of a share
    double inv;          // 1 / per
    int x;               // shares that the line is cut into
    int cnt, each;       // parts: of the lane's unit, steps of one

    __device__ AttnLine(const AttnArgs& a_, const AttnPlan& pl_, int64_t* lds) : a(a_), pl(pl_), ends(lds), R(pl_.units) {
        if (pl.per_row) {
            total = x = R;
            per = 1;
            inv = 1.0;
            return;
        }
        if (R <= 64) {
            const int lane = threadIdx.x & 63;
            const AttnSpan s = lane < R ? attn_span<SPANS>(a, lane) : AttnSpan{-1, 0, 0};
            len = s.n;
            gap = s.gap;
            seq = s.seq;
            upto = wave_scan(len < 0 ? 0 : attn_steps(len));  // (64 rows of 2^30 positions: 2^29)
            total = __builtin_amdgcn_readlane(upto, 63);
        } else {
            // wave w: rows 64 w .. 64 w + 63 and every 256 behind them
            __shared__ int block[kAttnPlanRows / 64];
            const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
            for (int r = wave * 64; r < R; r += kAttnThreads) {
                const int up = wave_scan(r + lane < R ? attn_steps(attn_span<SPANS>(a, r + lane).n) : 0);
                if (r + lane < R) ends[r + lane] = up;
                if (lane == 63) block[r / 64] = up;
            }
            __syncthreads();
            total = 0;
            for (int r = 0; r < R; r += 64) {
                if ((r / 64) % kAttnWaves == wave && r + lane < R) ends[r + lane] += total;
                total += block[r / 64];
            }
            __syncthreads();
        }
        // (whole numbers below 2^53: a quotient in doubles is off by one at most)
        per = max((int64_t)1, (int64_t)((double)total * pl.inv_shares));
        if ((per - 1) * pl.shares >= total) --per;
        while (per * pl.shares < total) ++per;
        if (PARTS && pl.parts) {
            const int steps = len < 0 ? 0 : attn_steps(len);
            // (at most 2^23 steps of a unit, and longer parts at most twice as long)
            for (int p = (int)per;; p += max(1, p / 8)) {
                cnt = ceil_quot(steps, p);
                if (__builtin_amdgcn_readlane(wave_scan(cnt), 63) <= pl.shares) break;
            }
            each = cnt ? ceil_quot(steps, cnt) : 1;
            cnt = ceil_quot(steps, each);
            upto = wave_scan(cnt);
            total = x = __builtin_amdgcn_readlane(upto, 63);
            per = 1;
            inv = 1.0;
            return;
        }
        // (at most 2048 shares: 2^-20 of a quotient is enough)
        inv = __builtin_amdgcn_rcp((double)per);
        x = share_of(total - 1) + 1;
    }
    // n / d rounded up, n and d up to 2^23, the quotient up to 2^20.
    static __device__ int ceil_quot(int n, int d) {
        const int m = n + d - 1;
        int q = (int)((float)m * __builtin_amdgcn_rcpf((float)d));
        q -= (int64_t)q * d > m;
        return q + ((int64_t)(q + 1) * d <= m);
    }
    // First step of share b; the share that holds a step.
    __device__ int64_t begin(int b) const { return min(b * per, total); }
    __device__ int share_of(int64_t step) const {
        int b = (int)((double)step * inv);
        b -= b * per > step;
        return b + ((b + 1) * per <= step);
    }
    // First unit that ends after `step`.
    __device__ int row_at(int64_t step) const {
        if (pl.per_row) return (int)step;
        if (R <= 64) return __builtin_amdgcn_readfirstlane(__builtin_ctzll(__ballot(step < upto)));
        int lo = 0, hi = (int)R - 1;
        while (lo < hi) {
            const int mid = (lo + hi) / 2;
            if (step < ends[mid]) hi = mid;
            else lo = mid + 1;
        }
        return __builtin_amdgcn_readfirstlane(lo);
    }
    // Unit r, from step `from` (of the line) up to step `to`.
    __device__ AttnSeg segment(int r, int64_t from, int64_t to, int64_t* end) const {
        AttnSeg g;
        g.row = r;
        if (pl.per_row) {
            const AttnSpan s = attn_span<SPANS>(a, r);
            g.n = s.n;
            g.gap = s.gap;
            g.seq = s.seq;
            g.p0 = 0;
            g.p1 = g.n;
            g.nc = 1;
            g.slot = 2 * (int64_t)r;  // (share r + row r)
            *end = r + 1;
            return g;
        }
        int64_t first;
        if (PARTS && pl.parts) {
            const int n = __builtin_amdgcn_readlane(each, r) * kAttnStep;
            g.n = __builtin_amdgcn_readlane(len, r);
            g.gap = __builtin_amdgcn_readlane(gap, r);
            g.seq = __builtin_amdgcn_readlane(seq, r);
            g.nc = __builtin_amdgcn_readlane(cnt, r);
            first = __builtin_amdgcn_readlane(upto, r) - g.nc;
            g.p0 = (int)(from - first) * n;
            g.p1 = min(g.p0 + n, g.n);
            g.slot = first + r;
            *end = to;
            return g;
        }
        if (R <= 64) {
            g.n = __builtin_amdgcn_readlane(len, r);
            g.gap = __builtin_amdgcn_readlane(gap, r);
            // (rows that are units by themselves: a load, 0.05 us less than a lane's)
            if constexpr (SPANS) g.seq = __builtin_amdgcn_readlane(seq, r);
            else g.seq = a.seq ? a.seq[r] : r;
            *end = __builtin_amdgcn_readlane(upto, r);
            first = *end - attn_steps(g.n);
        } else {
            const AttnSpan s = attn_span<SPANS>(a, r);
            g.n = s.n;
            g.gap = s.gap;
            g.seq = s.seq;
            *end = ends[r];
            first = r ? ends[r - 1] : 0;
        }
        g.p0 = (int)(max(from, first) - first) * kAttnStep;
        g.p1 = min((int)(min(to, *end) - first) * kAttnStep, g.n);
        g.nc = share_of(*end - 1) - share_of(first) + 1;
        g.slot = share_of(first) + r;
        return g;
    }
};

__device__ __forceinline__ float rows_max(float v) {  // over the lanes l, l ^ 16, l ^ 32, l ^ 48
    auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float rows_sum(float v) {
    auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// Over the wave, in every lane.
__device__ __forceinline__ float wave_max(float v) {
    for (int o = 1; o < 16; o <<= 1) v = fmaxf(v, __shfl_xor(v, o));
    return rows_max(v);
}
__device__ __forceinline__ float wave_sum(float v) {
    for (int o = 1; o < 16; o <<= 1) v += __shfl_xor(v, o);
    return rows_sum(v);
}
__device__ __forceinline__ float pow2(float v) { return __builtin_amdgcn_exp2f(v); }

// Two floats at device scope.
__device__ __forceinline__ void st2_device(float* p, float x, float y) {
    const unsigned long long v = ((unsigned long long)__float_as_uint(y) << 32) | __float_as_uint(x);
    __hip_atomic_store(reinterpret_cast<unsigned long long*>(p), v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float2 ld2_device(const float* p) {
    const unsigned long long v = __hip_atomic_load(reinterpret_cast<const unsigned long long*>(p), __ATOMIC_RELAXED,
                                                   __HIP_MEMORY_SCOPE_AGENT);
    return float2{__uint_as_float((unsigned)v), __uint_as_float((unsigned)(v >> 32))};
}

__device__ __forceinline__ float row_lse(float m, float l) {
    return l == 0.0f ? -INFINITY : (m + log2f(l)) * 0.69314718056f;
}

constexpr int kJoinGroup = 32;

// Joins `cnt` (at most 64) segments, in every `every`-th slot from slot0, for
// the columns 0 .. nh - 1: into their rows' results (last), or into slot0.
// A wave adds up one head's columns, a pair a lane; the segments' maxima and
// sums are a lane's each; with one or two heads the waves share the segments.
// Bound by the latency of device-scope loads: the first segments' columns are
// requested together with the statistics that weigh them.  where(h): the row
// and the query head of column h.
struct AttnPlace {
    int row, head;
};
template <int DP, typename Where>
__device__ void attention_join(const AttnArgs& a, const AttnPlan& pl, Where where, int64_t slot0, int every, int cnt,
                               bool last, int nh, float* scratch) {
    constexpr int NK = DP > 128 ? 2 : 1, N = 16;  // pairs of a lane, segments in flight
    const int D = a.c.D, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int64_t first = slot0 * pl.hy + blockIdx.y, step = (int64_t)every * pl.hy * 16 * pl.dp;
    const int share = nh == 1 ? 4 : (nh == 2 ? 2 : 1), part = wave & (share - 1);
#pragma unroll 1
    for (int hb = 0; hb < nh; hb += kAttnWaves / share) {
        const int h = min(hb + wave / share, nh - 1);  // (a head too many: a repeat, not written)
        float* o = pl.part_o + (first * 16 + h) * pl.dp;
        float* ml = pl.part_ml + (first * 16 + h) * 2;
        const float2 st = ld2_device(ml + (int64_t)min(lane, cnt - 1) * every * pl.hy * 32);
        float m = 0.0f, l = 0.0f, fc = 0.0f;  // fc: the factor of the lane's segment
        float2 v[NK];
#pragma unroll
        for (int k = 0; k < NK; ++k) v[k] = float2{0.0f, 0.0f};
#pragma unroll 1
        for (int c = part; c < cnt || c == part; c += N * share) {
            float2 x[N][NK];
#pragma unroll
            for (int i = 0; i < N; ++i)
#pragma unroll
                for (int k = 0; k < NK; ++k)
                    if (2 * lane + 128 * k < D)
                        x[i][k] = ld2_device(o + min(c + i * share, cnt - 1) * step + 2 * lane + 128 * k);
            if (c == part) {
                const float mc = lane < cnt ? st.x : -INFINITY;
                m = wave_max(mc);
                fc = pow2(mc - (m == -INFINITY ? 0.0f : m));
                l = wave_sum(lane < cnt ? st.y * fc : 0.0f);
            }
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int ci = c + i * share;
                const float f = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(fc), min(ci, 63)));
#pragma unroll
                for (int k = 0; k < NK; ++k)
                    if (ci < cnt && 2 * lane + 128 * k < D) {
                        v[k].x += f * x[i][k].x;
                        v[k].y += f * x[i][k].y;
                    }
            }
        }
        if (share > 1) {  // scratch [4][256]
            __syncthreads();
#pragma unroll
            for (int k = 0; k < NK; ++k) {
                scratch[wave * 256 + 2 * lane + 128 * k] = v[k].x;
                scratch[wave * 256 + 2 * lane + 128 * k + 1] = v[k].y;
            }
            __syncthreads();
            if (part == 0)
                for (int w = 1; w < share; ++w)
#pragma unroll
                    for (int k = 0; k < NK; ++k) {
                        v[k].x += scratch[(wave + w) * 256 + 2 * lane + 128 * k];
                        v[k].y += scratch[(wave + w) * 256 + 2 * lane + 128 * k + 1];
                    }
        }
        if (hb + wave / share >= nh || part) continue;
        if (!last) {
            // (the wave itself has read what lay there)
#pragma unroll
            for (int k = 0; k < NK; ++k)
                if (2 * lane + 128 * k < D) st2_device(o + 2 * lane + 128 * k, v[k].x, v[k].y);
            if (lane == 0) st2_device(ml, m, l);
            continue;
        }
        const AttnPlace w = where(h);
        float* to = a.out + w.row * a.ldo + (int64_t)w.head * D;
#pragma unroll
        for (int k = 0; k < NK; ++k) {
            const int d = 2 * lane + 128 * k;
            if (d < D) to[d] = l == 0.0f ? 0.0f : v[k].x / l;
            if (d + 1 < D) to[d + 1] = l == 0.0f ? 0.0f : v[k].y / l;
        }
        if (lane == 0) {
            const int64_t at = (int64_t)w.row * a.hq + w.head;
            if (a.lse) a.lse[at] = row_lse(m, l);
            if (pl.ml) {
                pl.ml[2 * at] = m;
                pl.ml[2 * at + 1] = l;
            }
        }
    }
}

// Counts one of `of` results, stored by this workgroup, and says whether it
// was the last.  (The count wraps to zero by itself, for the next call.)
__device__ __forceinline__ bool attention_count(unsigned* count, int of, int* lds_last) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // every store has arrived
    __syncthreads();
    if (threadIdx.x == 0) *lds_last = atomicInc(count, (unsigned)of - 1) == (unsigned)of - 1;
    __syncthreads();
    return *lds_last;
}

// Bytes of the plan's arrays in one workspace; `parts`: whether a unit may be in
// more than one segment.
inline size_t place_attention(const AttnArgs& a, AttnPlan* pl, bool parts, char* base) {
    size_t at = 0;
    auto take = [&](size_t floats) {
        float* p = reinterpret_cast<float*>(base + at);
        at += (floats * 4 + 255) / 256 * 256;
        return p;
    };
    const size_t slots = (size_t)pl->shares + (size_t)pl->units;
    if (parts) {
        pl->part_ml = take(slots * pl->hy * 32);
        pl->part_o = take(slots * pl->hy * 16 * pl->dp);
    }
    if (a.accumulate) {
        pl->ml = take((size_t)a.R * a.hq * 2);
        pl->s = take((size_t)a.R * a.hq * pl->cap);
    }
    return at;
}

// The plan of units of `rows` rows, `resident` workgroups per compute unit.
inline AttnPlan plan_attention(const AttnArgs& a, int cus, int rows, int resident) {
    AttnPlan pl;
    const int G = a.hq / a.c.hkv;
    pl.part_o = pl.part_ml = pl.s = pl.ml = nullptr;
    pl.count = pl.tops = nullptr;
    pl.dp = (a.c.D + 1) / 2 * 2;
    pl.tiles = (G + 15) / 16;
    pl.hy = a.c.hkv * pl.tiles;
    const int64_t cap = (int64_t)a.c.max_pages * a.c.page;
    const int64_t each = (a.tokens + rows - 1) / rows;  // units of a sequence's rows
    pl.cap = (std::min(cap, (int64_t)a.window + a.sink) + 31) / 32 * 32;
    pl.units = (int)(rows == 1 ? a.R : a.R / a.tokens * each);
    pl.per_row = a.call_rows / a.tokens * each > kAttnPlanRows;
    const int64_t steps = pl.units * std::max<int64_t>(1, (cap + kAttnStep - 1) / kAttnStep);
    pl.shares = (int)std::min(steps, std::max<int64_t>(1, (int64_t)resident * cus / pl.hy));
    pl.shares = std::min(pl.shares, 64 * kJoinGroup);  // (as many as two levels join)
    if (pl.per_row) pl.shares = pl.units;
    pl.inv_shares = 1.0 / (double)pl.shares;
    pl.parts = false;
    return pl;
}
inline bool attention_splits(const AttnArgs& a, const AttnPlan& pl) {
    return !pl.per_row && (int64_t)a.c.max_pages * a.c.page > kAttnStep;
}
// Its counters, and where they lie.
inline size_t attention_counters(const AttnArgs& a, const AttnPlan& pl) {
    return attention_splits(a, pl) ? ((size_t)pl.shares + 2 * (size_t)pl.units) * pl.hy * sizeof(unsigned) : 0;
}
inline void attention_memory(const AttnArgs& a, AttnPlan* pl, void* ws, void* counters) {
    (void)place_attention(a, pl, attention_splits(a, *pl), static_cast<char*>(ws));
    pl->count = static_cast<unsigned*>(counters);
    pl->tops = pl->count + ((size_t)pl->shares + (size_t)pl->units) * pl->hy;
}

}  // namespace xt
