// The paged key-value cache's append (rotary embedding, rounding, scatter)
// and the attention of one token per row over it.
#include <algorithm>

#include "xtern_cache.h"

namespace xt {

// ---------------------------------------------------------------------------
// Append
// ---------------------------------------------------------------------------
// With h = rot / 2, element i < h of a rotated head becomes
//   x[i] cos - x[i + h] sin,   element i + h   x[i + h] cos + x[i] sin
// (cos, sin: row `pos`, column i of the tables); elements from rot on, and
// values, are copied.  One workgroup per row, W neighbouring pairs (or copied
// elements) a thread: four where the head size and h are multiples of four, two
// where they are even (no alignment is needed for that).  Large calls are bound
// by HBM: 4096 rows of 32 + 2 x 8 heads of 128 into f16 pages take 38 us, 4.9
// TB/s (47 us an element at a time); small ones by the launch, 3.4 us.
template <typename T, int W>
struct AppendVec {
    typedef T V __attribute__((ext_vector_type(W)));
    typedef V U __attribute__((aligned(sizeof(T))));
    static __device__ __forceinline__ V get(const T* p) { return *reinterpret_cast<const U*>(p); }
    static __device__ __forceinline__ void put(T* p, V v) { *reinterpret_cast<U*>(p) = v; }
};

template <int DT, int W>
__global__ __launch_bounds__(256) void kv_append_kernel(AppendArgs a) {
    typedef Elem<DT> E;
    typedef typename E::T T;
    typedef AppendVec<float, W> F;
    typedef typename F::V VF;
    const int64_t r = blockIdx.x;
    const KvView& c = a.c;
    const int slot = a.slots[r];
    const int sq = a.seq ? a.seq[r] : (int)r;
    const int pos = a.cos ? a.pos[r] : 0;
    int pg = -1;
    if (slot >= 0 && slot < (int64_t)c.max_pages * c.page && (unsigned)sq < (unsigned)c.nseq &&
        (!a.cos || (pos >= 0 && pos < a.rope_rows)))
        pg = kv_page(c, sq, slot);
    if (a.lengths && threadIdx.x == 0) a.lengths[r] = pg < 0 ? 0 : slot + 1;
    if (pg < 0) return;
    const int half = a.cos ? a.rot / 2 : 0, per = (c.D - half) / W;  // work items of one rotated head
    const int nq = (a.q ? a.hq : 0) * per, nk = c.hkv * per, vals = c.D / W, nv = c.hkv * vals;
    const int64_t at = kv_offset(c, pg, slot, 0);
    T* kc = static_cast<T*>(c.k) + at;
    T* vc = static_cast<T*>(c.v) + at;
    auto store = [&](T* p, VF v) {
        typename AppendVec<T, W>::V y;
#pragma unroll
        for (int x = 0; x < W; ++x) y[x] = E::put(v[x]);
        AppendVec<T, W>::put(p, y);
    };
    for (int i = threadIdx.x; i < nq + nk + nv; i += blockDim.x) {
        if (i >= nq + nk) {
            const int j = i - nq - nk, h = fast_quot(j, a.by_vals), d = (j - h * vals) * W;
            store(vc + h * c.sh + d, F::get(a.v + r * a.ldv + (int64_t)j * W));
            continue;
        }
        const bool isq = i < nq;
        const int j = isq ? i : i - nq, h = fast_quot(j, a.by_per), e = (j - h * per) * W;
        const float* x = (isq ? a.q + r * a.ldq : a.k + r * a.ldk) + (int64_t)h * c.D;
        float* qo = a.qo + r * a.ldqo + (int64_t)h * c.D;
        T* ko = kc + h * c.sh;
        if (e < half) {
            const VF cs = F::get(a.cos + (int64_t)pos * half + e), sn = F::get(a.sin + (int64_t)pos * half + e);
            const VF x0 = F::get(x + e), x1 = F::get(x + e + half);
            VF y0, y1;
#pragma unroll
            for (int k = 0; k < W; ++k) {
                y0[k] = x0[k] * cs[k] - x1[k] * sn[k];
                y1[k] = x1[k] * cs[k] + x0[k] * sn[k];
            }
            if (isq) {
                F::put(qo + e, y0);
                F::put(qo + e + half, y1);
            } else {
                store(ko + e, y0);
                store(ko + e + half, y1);
            }
        } else {
            const VF y = F::get(x + e + half);
            if (isq) F::put(qo + e + half, y);
            else store(ko + e + half, y);
        }
    }
    if (c.score)
        for (int h = threadIdx.x; h < c.hkv; h += blockDim.x)
            c.score[((int64_t)pg * c.hkv + h) * c.page + kv_slot(c, slot)] = 0.0f;
}

template <int DT>
hipError_t launch_append(AppendArgs& a, hipStream_t s) {
    const int half = a.cos ? a.rot / 2 : 0, odd = a.c.D | half, w = odd % 2 ? 1 : (odd % 4 ? 2 : 4);
    a.by_per = fast_div((a.c.D - half) / w);
    a.by_vals = fast_div(a.c.D / w);
    if (w == 4)
        kv_append_kernel<DT, 4><<<(unsigned)a.R, 256, 0, s>>>(a);
    else if (w == 2)
        kv_append_kernel<DT, 2><<<(unsigned)a.R, 256, 0, s>>>(a);
    else
        kv_append_kernel<DT, 1><<<(unsigned)a.R, 256, 0, s>>>(a);
    return hipGetLastError();
}

hipError_t launch_kv_append(int dtype, AppendArgs a, hipStream_t s) {
    switch (dtype) {
        case XT_F32: return launch_append<XT_F32>(a, s);
        case XT_F16: return launch_append<XT_F16>(a, s);
        default: return launch_append<XT_BF16>(a, s);
    }
}

// ---------------------------------------------------------------------------
// Attention
// ---------------------------------------------------------------------------
// For each row and query head, over the positions j < length whose page
// exists: s_j = scale q.k_j, m = max s, l = sum exp(s_j - m),
// out = sum exp(s_j - m) v_j / l, lse = m + ln l.  A row without positions
// (or whose every s_j is -inf) gives zeros and lse = -inf.
//
// The cache is read once, so HBM bounds it: a position of one key-value head
// is 4 D bytes (16-bit types) for 4 D G operations, G query heads a group.
// The matrix cores do the products with the query heads of a group as their
// 16 columns, transposed so that nothing moves between lanes:
//   S^T = K Q^T: the lane that holds column h (lane & 15) gets S of head h for
//     four positions per 16 (rows 4 g .. 4 g + 3, g = lane >> 4);
//   O^T = V^T P^T: the sum runs over positions in any order, so the lane's own
//     P values are its operand as they are; V^T's operand wants, per lane, one
//     column of eight positions, which the lane loads as eight row pieces and
//     transposes in registers (v_perm);
//   the softmax factors of a head are then the lane's own, also for O^T.
// 16-bit caches: q and p in f32 are split into three bf16 or f16 pieces (f16's
// raised against its short range), whose products with k, v the 16-bit MFMA
// adds up in f32: the matrix cores have that to spare (at D = 128, 48
// instructions of 16 cycles per 32 positions against the 6700 cycles that their
// 16 KB take a SIMD at 6 TB/s).  f32 caches take the f32 MFMA.
// Measured (kernel time): 64 rows of up to 8192 positions, 32 query and 8 kv
// heads of 128, f16, 186 us (5.8 TB/s of cache); 131072 positions of one row,
// bf16, 95 us (5.6 TB/s); 700 positions of 20 and 5 heads 11.5 us, where the
// chain of dependent loads (lengths, table, keys, then the join's) counts.

typedef float v4f __attribute__((ext_vector_type(4)));
typedef int v2i __attribute__((ext_vector_type(2)));
typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
// (rows may start at any element: the hardware loads unaligned vectors)
typedef v4i v4iu __attribute__((aligned(2)));
typedef v2i v2iu __attribute__((aligned(2)));
typedef v4f v4fu __attribute__((aligned(4)));

constexpr int kAttnThreads = 256;
constexpr int kAttnWaves = kAttnThreads / 64;
constexpr int kAttnStep = 128;       // positions: the unit of the split
constexpr int kAttnPlanRows = 1024;  // rows whose work is split by its total

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
    int64_t cap;     // positions of a row of s, a multiple of 32
    int hy;          // workgroups per share: kv heads x tiles of 16 query heads
    int tiles;       // of 16 query heads per kv head
    int shares;      // at most
    bool per_row;
};

// A row's part of the line, and of it what one share covers.
struct AttnSeg {
    int row, n, p0, p1;  // positions [p0, p1) of n
    int nc;              // segments of the row
    int64_t slot;        // of its first one
};

__device__ __forceinline__ int attn_len(const AttnArgs& a, int64_t r) {
    const int sq = a.seq ? a.seq[r] : (int)r;
    return (unsigned)sq < (unsigned)a.c.nseq ? kv_length(a.c, a.lengths[r]) : 0;
}
__device__ __forceinline__ int attn_steps(int len) { return max(1, (len + kAttnStep - 1) / kAttnStep); }

// The line as every wave of the workgroup sees it: 64 rows, a lane each, in
// registers (no barrier), or the rows' ends in LDS.
struct AttnLine {
    const AttnArgs& a;
    const AttnPlan& pl;
    int len, upto;       // the lane's row (R <= 64)
    int64_t* ends;       // LDS, [R] (R > 64)
    int64_t total;       // steps
    int64_t per;         // steps of a share
    double inv;          // 1 / per
    int x;               // shares that the line is cut into

    __device__ AttnLine(const AttnArgs& a_, const AttnPlan& pl_, int64_t* lds) : a(a_), pl(pl_), ends(lds) {
        if (pl.per_row) {
            total = x = (int)a.R;
            per = 1;
            inv = 1.0;
            return;
        }
        if (a.R <= 64) {
            const int lane = threadIdx.x & 63;
            len = lane < a.R ? attn_len(a, lane) : -1;
            upto = wave_scan(len < 0 ? 0 : attn_steps(len));  // (64 rows of 2^30 positions: 2^29)
            total = __builtin_amdgcn_readlane(upto, 63);
        } else {
            // wave w: rows 64 w .. 64 w + 63 and every 256 behind them
            __shared__ int block[kAttnPlanRows / 64];
            const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
            for (int r = wave * 64; r < a.R; r += kAttnThreads) {
                const int up = wave_scan(r + lane < a.R ? attn_steps(attn_len(a, r + lane)) : 0);
                if (r + lane < a.R) ends[r + lane] = up;
                if (lane == 63) block[r / 64] = up;
            }
            __syncthreads();
            total = 0;
            for (int r = 0; r < a.R; r += 64) {
                if ((r / 64) % kAttnWaves == wave && r + lane < a.R) ends[r + lane] += total;
                total += block[r / 64];
            }
            __syncthreads();
        }
        // (whole numbers below 2^53: a quotient in doubles is off by one at most)
        per = max((int64_t)1, (int64_t)((double)total / (double)pl.shares));
        while (per * pl.shares < total) ++per;
        inv = 1.0 / (double)per;
        x = share_of(total - 1) + 1;
    }
    // First step of share b; the share that holds a step.
    __device__ int64_t begin(int b) const { return min(b * per, total); }
    __device__ int share_of(int64_t step) const {
        int b = (int)((double)step * inv);
        b -= b * per > step;
        return b + ((b + 1) * per <= step);
    }
    // First row that ends after `step`.
    __device__ int row_at(int64_t step) const {
        if (pl.per_row) return (int)step;
        if (a.R <= 64) return __builtin_amdgcn_readfirstlane(__builtin_ctzll(__ballot(step < upto)));
        int lo = 0, hi = (int)a.R - 1;
        while (lo < hi) {
            const int mid = (lo + hi) / 2;
            if (step < ends[mid]) hi = mid;
            else lo = mid + 1;
        }
        return __builtin_amdgcn_readfirstlane(lo);
    }
    // Row r, from step `from` (of the line) up to step `to`.
    __device__ AttnSeg segment(int r, int64_t from, int64_t to, int64_t* end) const {
        AttnSeg g;
        g.row = r;
        if (pl.per_row) {
            g.n = attn_len(a, r);
            g.p0 = 0;
            g.p1 = g.n;
            g.nc = 1;
            g.slot = 2 * (int64_t)r;  // (share r + row r)
            *end = r + 1;
            return g;
        }
        int64_t first;
        if (a.R <= 64) {
            g.n = __builtin_amdgcn_readlane(len, r);
            *end = __builtin_amdgcn_readlane(upto, r);
            first = *end - attn_steps(g.n);
        } else {
            g.n = attn_len(a, r);
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

// Pieces of an f32 operand x: the first is x rounded, each further one STEP
// times what the one before left of it.
template <int DT> struct Split;
template <> struct Split<XT_BF16> {
    typedef v8bf V;
    static constexpr int N = 3;
    static constexpr float STEP = 1.0f;
    static constexpr float P = 1.0f;  // scale of the probabilities
    static __device__ __forceinline__ v4f mfma(V a, V b, v4f c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
    }
};
template <> struct Split<XT_F16> {
    typedef v8h V;
    static constexpr int N = 3;
    // f16 has 11 bits, and none below 2^-24: raised by 2^11, the next piece holds
    // the next 11 bits, and what three pieces leave is below 2^-47.  With p <= 1
    // as 2^14 p, weights down to 2^-37 of the row's largest keep all 24 bits, and
    // smaller ones are off by 2^-61 of it at most.  (Two pieces without the raise,
    // steps of 2^-39: weights of 2^-26 had lost their last 11 bits; heads of 64 /
    // 128 / 256 took 53 / 182 / 172 us and take 55 / 186 / 184.)
    static constexpr float STEP = 2048.0f;
    static constexpr float P = 16384.0f;
    static __device__ __forceinline__ v4f mfma(V a, V b, v4f c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
    }
};
template <int DT>
__device__ __forceinline__ void split8(const float* x, typename Split<DT>::V* out) {
    typedef typename Elem<DT>::T T;
    float r[8];
    for (int i = 0; i < 8; ++i) r[i] = x[i];
#pragma unroll
    for (int n = 0; n < Split<DT>::N; ++n)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const T p = (T)r[i];
            out[n][i] = p;
            r[i] = (r[i] - (float)p) * Split<DT>::STEP;
        }
}

// The shape of a workgroup's registers: DP the padded head size (64, 128, 256).
template <int DT, int DP>
struct AttnShape {
    static constexpr bool F32 = DT == XT_F32;
    static constexpr int ES = F32 ? 4 : 2;
    static constexpr int TK = F32 ? 16 : 32;       // positions per tile of a wave
    static constexpr int NT = TK / 16;
    static constexpr int KU = 16 / ES;             // elements of a key load
    static constexpr int KS = DP / (4 * KU);       // key loads per 16 positions
    static constexpr int NJ = TK / 4;              // positions of a lane's V piece
    static constexpr int UE = DP / 16 < KU ? DP / 16 : KU;  // elements of a value load
    static constexpr int NU = DP / 16 / UE;        // value loads per position
};

// One chunk [p0, p1) of a row for the heads h0 .. h0 + nh - 1, in plain f32
// operations: what the matrix cores' split operands cannot give (infinities
// and NaN among the inputs, sums past f32's range in a piece) and head sizes
// below one load.  256 positions at a time, one head after the other; the sums
// go where the matrix cores' would be.
template <int DT>
__device__ void attn_plain(const AttnArgs& a, const AttnPlan& pl, const AttnSeg& it, int hk, int h0, int nh,
                           float scale2, float* lds_o, float* lds_ml, int ldo) {
    typedef Elem<DT> E;
    const KvView& c = a.c;
    const int t = threadIdx.x, sq = a.seq ? a.seq[it.row] : it.row;
    __shared__ float sp[kAttnThreads];
    __shared__ int64_t so[kAttnThreads];
    __shared__ float sm[kAttnWaves];
    const typename E::T* kc = static_cast<const typename E::T*>(c.k);
    const typename E::T* vc = static_cast<const typename E::T*>(c.v);
    for (int h = 0; h < nh; ++h) {
        const float* q = a.q + it.row * a.ldq + (int64_t)(h0 + h) * c.D;
        float m = -INFINITY, l = 0.0f, o = 0.0f;
        for (int p0 = it.p0; p0 < it.p1; p0 += kAttnThreads) {
            const int p = p0 + t, pg = p < it.p1 ? kv_page(c, sq, p) : -1;
            const int64_t off = pg < 0 ? -1 : kv_offset(c, pg, p, hk);
            float s = -INFINITY;
            if (off >= 0) {
                float acc = 0.0f;
                for (int d = 0; d < c.D; ++d) acc += q[d] * E::get(kc[off + d]);
                s = acc * scale2;
            }
            if (pl.s && p < it.p1) pl.s[((int64_t)it.row * a.hq + h0 + h) * pl.cap + p] = s;
            float v = s;
            for (int x = 32; x; x >>= 1) v = fmaxf(v, __shfl_xor(v, x));
            __syncthreads();
            if ((t & 63) == 0) sm[t >> 6] = v;
            so[t] = off;
            __syncthreads();
            const float mn = fmaxf(m, fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3])));
            const float base = mn == -INFINITY ? 0.0f : mn;
            const float f = pow2(m - base);
            sp[t] = off < 0 ? 0.0f : pow2(s - base);
            m = mn;
            l *= f;
            o *= f;
            __syncthreads();
            const int cnt = min(kAttnThreads, it.p1 - p0);
            for (int j = 0; j < cnt; ++j)
                if (so[j] >= 0) {
                    l += sp[j];
                    if (t < c.D) o += sp[j] * E::get(vc[so[j] + t]);
                }
            __syncthreads();
        }
        if (t < c.D) lds_o[h * ldo + t] = o;
        if (t == 0) {
            lds_ml[h] = m;
            lds_ml[16 + h] = l;
        }
    }
    __syncthreads();
}

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
// the heads h0 .. h0 + nh - 1: into the row's results (last), or into slot0.
// A wave adds up one head's columns, a pair a lane; the segments' maxima and
// sums are a lane's each; with one or two heads the waves share the segments.
// Bound by the latency of device-scope loads: the first segments' columns are
// requested together with the statistics that weigh them.
template <int DP>
__device__ void attention_join(const AttnArgs& a, const AttnPlan& pl, int row, int64_t slot0, int every, int cnt,
                               bool last, int h0, int nh, float* scratch) {
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
        float* to = a.out + row * a.ldo + (int64_t)(h0 + h) * D;
#pragma unroll
        for (int k = 0; k < NK; ++k) {
            const int d = 2 * lane + 128 * k;
            if (d < D) to[d] = l == 0.0f ? 0.0f : v[k].x / l;
            if (d + 1 < D) to[d + 1] = l == 0.0f ? 0.0f : v[k].y / l;
        }
        if (lane == 0) {
            const int64_t at = (int64_t)row * a.hq + h0 + h;
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

template <int DT, int DP>
__global__ __launch_bounds__(kAttnThreads, DP == 256 ? 1 : (DP == 128 ? 2 : 3)) void attention_kernel(AttnArgs a, AttnPlan pl,
                                                                                   float scale2) {
    typedef AttnShape<DT, DP> S;
    typedef Elem<DT> E;
    typedef typename E::T T;
    const KvView& c = a.c;
    constexpr int kLdsRow = DP + 4;  // floats; the pad keeps heads apart in the banks
    __shared__ v4i lds_mem[kAttnWaves * 16 * kLdsRow / 4];
    v4i* lds_q = lds_mem;                                // the queries, then
    float* lds_o = reinterpret_cast<float*>(lds_mem);    // the waves' sums
    __shared__ float lds_ml[kAttnWaves][2][16];
    __shared__ int64_t lds_off[kAttnWaves][2][32];
    __shared__ int lds_last;
    __shared__ int64_t lds_ends[kAttnPlanRows];
    const int hk = blockIdx.y / pl.tiles, G = a.hq / c.hkv;
    const int h0 = hk * G + (blockIdx.y % pl.tiles) * 16, nh = min(16, hk * G + G - h0);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const AttnLine line(a, pl, lds_ends);
    if ((int)blockIdx.x >= line.x) return;
    int64_t at = line.begin(blockIdx.x);
    const int64_t to_step = line.begin(blockIdx.x + 1);
    for (int r = line.row_at(at); at < to_step; ++r) {
        int64_t row_end;
        const AttnSeg it = line.segment(r, at, to_step, &row_end);
        at = row_end;
        // (opaque to the compiler: it would keep every index that follows from
        // them in registers from segment to segment, and spill)
        int D = c.D, lane = threadIdx.x & 63;
        asm volatile("" : "+s"(D), "+v"(lane));
        const int n = lane & 15, g = lane >> 4;
        const bool fast = D >= S::KU;
        const int sq = a.seq ? a.seq[r] : r;
        const int ntiles = it.p1 > it.p0 ? (it.p1 - it.p0 + S::TK - 1) / S::TK : 0;

        float m = -INFINITY, l = 0.0f, qs = scale2;
        v4f o[S::NU * S::UE];
    #pragma unroll
        for (int i = 0; i < S::NU * S::UE; ++i) o[i] = v4f{0.0f, 0.0f, 0.0f, 0.0f};

        if (fast && ntiles > 0) {
            const T* kc = static_cast<const T*>(c.k);
            const T* vc = static_cast<const T*>(c.v);
            // byte offsets of the lane's pieces in a key's and a value's row
            int kd[S::KS], vd[S::NU];
    #pragma unroll
            for (int s = 0; s < S::KS; ++s) kd[s] = min(S::KU * (4 * s + g), D - S::KU);
    #pragma unroll
            for (int u = 0; u < S::NU; ++u) vd[u] = min(16 * S::UE * u + S::UE * n, D - S::UE);

            v4i kr[S::NT][S::KS];
            v4i vr[S::NJ][S::NU];
            // Row offsets of a tile's positions, one lane each, through the wave's
            // LDS; -1: no position there (masked, read from offset 0)
            auto entry = [&](int i) {  // the lane's table entry of tile i
                const int p = it.p0 + i * S::TK + (lane & (S::TK - 1));
                return p < it.p1 ? c.table[(int64_t)sq * c.ldt + kv_page_of(c, p)] : -1;
            };
            auto offsets = [&](int i, int e) {
                const int p = it.p0 + i * S::TK + (lane & (S::TK - 1));
                const int64_t off = (unsigned)e < (unsigned)c.num_pages ? kv_offset(c, e, p, hk) : -1;
                if (lane < S::TK) lds_off[wave][(i / kAttnWaves) & 1][lane] = off;
                return __ballot(off < 0) == 0;
            };
            auto load_k = [&](int i) {
                const int64_t* of = lds_off[wave][(i / kAttnWaves) & 1];
    #pragma unroll
                for (int t = 0; t < S::NT; ++t) {
                    const T* row = kc + max(of[16 * t + n], (int64_t)0);
    #pragma unroll
                    for (int s = 0; s < S::KS; ++s) kr[t][s] = *reinterpret_cast<const v4iu*>(row + kd[s]);
                }
            };
            // (16 lanes read a value row from end to end, so its lines need not
            // stay in the caches: 64 ragged rows 199 -> 180 us, 131072 positions
            // 105 -> 95.5.  A key row's lines are read by several loads: there
            // the hint costs up to a fifth where rows do not end with lines.)
            auto load_v = [&](int i) {
                const int64_t* of = lds_off[wave][(i / kAttnWaves) & 1];
    #pragma unroll
                for (int j = 0; j < S::NJ; ++j) {
                    const T* row = vc + max(of[16 * (j / 4) + 4 * g + j % 4], (int64_t)0);
    #pragma unroll
                    for (int u = 0; u < S::NU; ++u) {
                        if constexpr (S::UE * S::ES == 16) {
                            vr[j][u] = __builtin_nontemporal_load(reinterpret_cast<const v4iu*>(row + vd[u]));
                        } else {
                            const v2i x = __builtin_nontemporal_load(reinterpret_cast<const v2iu*>(row + vd[u]));
                            vr[j][u] = v4i{x[0], x[1], 0, 0};
                        }
                    }
                }
            };

            int next_e = entry(wave);
            const int after_e = entry(wave + kAttnWaves);
            // The query rows as the lanes' operands, to LDS (in registers they
            // would take 48 of 256 at D = 128), a wave every fourth piece: head
            // h0 + n, elements from min(KU (4 s + g), D - KU); where pieces
            // overlap (D no multiple of KU, or past D) the earlier one counts,
            // the later one holds zeros.
            const float* q = a.q + it.row * a.ldq + (int64_t)(h0 + (n < nh ? n : 0)) * D;
            auto q_load = [&](int s, float* x) {
                const int nom = S::KU * (4 * s + g), d = min(nom, D - S::KU);
#pragma unroll
                for (int i = 0; i < S::KU; i += 4) {
                    const v4f f = *reinterpret_cast<const v4fu*>(q + d + i);
#pragma unroll
                    for (int e = 0; e < 4; ++e) x[i + e] = n < nh && d + i + e >= nom ? f[e] : 0.0f;
                }
            };
            float up = 1.0f;
            if constexpr (DT == XT_F16) {
                // the row's largest element at 2^14 .. 2^15: the pieces then hold
                // every element down to 2^-37 of it, and 2^-61 of it of the others
                float mx = 0.0f;
#pragma unroll
                for (int s = 0; s < S::KS; ++s) {
                    float x[8];
                    q_load(s, x);
#pragma unroll
                    for (int i = 0; i < 8; ++i) mx = fmaxf(mx, fabsf(x[i]));
                }
                mx = rows_max(mx);
                int e = 0;
                if (mx > 0.0f && mx < INFINITY) {
                    (void)frexpf(mx, &e);
                    e = max(-100, min(100, 15 - e));
                }
                up = ldexpf(1.0f, e);
                qs = scale2 * ldexpf(1.0f, -e);
            }
#pragma unroll 1
            for (int s = wave; s < S::KS; s += kAttnWaves) {
                float x[S::KU];
                q_load(s, x);
                if constexpr (S::F32) {
                    lds_q[s * 64 + lane] = __builtin_bit_cast(v4i, v4f{x[0], x[1], x[2], x[3]});
                } else {
                    typename Split<DT>::V pieces[3];
#pragma unroll
                    for (int i = 0; i < 8; ++i) x[i] *= up;
                    split8<DT>(x, pieces);
#pragma unroll
                    for (int k = 0; k < Split<DT>::N; ++k)
                        lds_q[(s * Split<DT>::N + k) * 64 + lane] = __builtin_bit_cast(v4i, pieces[k]);
                }
            }
            bool full = false;
            if (wave < ntiles) {
                full = offsets(wave, next_e);
                next_e = after_e;
                load_k(wave);
                load_v(wave);
            }
            __syncthreads();
            for (int i = wave; i < ntiles; i += kAttnWaves) {
                asm volatile("" ::: "memory");  // (the queries stay in LDS)
                // S of the tile
                v4f sc[S::NT];
#pragma unroll
                for (int t = 0; t < S::NT; ++t) sc[t] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int s = 0; s < S::KS; ++s) {
                    if constexpr (S::F32) {
                        const v4f qv = __builtin_bit_cast(v4f, lds_q[s * 64 + lane]);
#pragma unroll
                        for (int x = 0; x < 4; ++x)
#pragma unroll
                            for (int t = 0; t < S::NT; ++t)
                                sc[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(__int_as_float(kr[t][s][x]), qv[x], sc[t],
                                                                             0, 0, 0);
                    } else if constexpr (Split<DT>::STEP == 1.0f) {
                        typedef typename Split<DT>::V V;
#pragma unroll
                        for (int x = Split<DT>::N - 1; x >= 0; --x) {
                            const V qv = __builtin_bit_cast(V, lds_q[(s * Split<DT>::N + x) * 64 + lane]);
#pragma unroll
                            for (int t = 0; t < S::NT; ++t)
                                sc[t] = Split<DT>::mfma(__builtin_bit_cast(V, kr[t][s]), qv, sc[t]);
                        }
                    }
                }
                if constexpr (DT == XT_F16) {  // a piece at a time, the last first
                    typedef typename Split<DT>::V V;
#pragma unroll
                    for (int x = Split<DT>::N - 1; x >= 0; --x) {
#pragma unroll
                        for (int s = 0; s < S::KS; ++s) {
                            const V qv = __builtin_bit_cast(V, lds_q[(s * Split<DT>::N + x) * 64 + lane]);
#pragma unroll
                            for (int t = 0; t < S::NT; ++t)
                                sc[t] = Split<DT>::mfma(__builtin_bit_cast(V, kr[t][s]), qv, sc[t]);
                        }
                        if (x)
#pragma unroll
                            for (int t = 0; t < S::NT; ++t) sc[t] *= 1.0f / Split<DT>::STEP;
                    }
                }
                // the next tile's keys, in flight under this tile's softmax and values
                const bool was_full = full;
                const int64_t* of = lds_off[wave][(i / kAttnWaves) & 1];
                if (i + kAttnWaves < ntiles) {
                    full = offsets(i + kAttnWaves, next_e);
                    next_e = entry(i + 2 * kAttnWaves);
                    load_k(i + kAttnWaves);
                }
                float p[S::NJ], mt = m;
    #pragma unroll
                for (int j = 0; j < S::NJ; ++j) {
                    p[j] = sc[j / 4][j % 4] * qs;
                    if (!was_full && of[16 * (j / 4) + 4 * g + j % 4] < 0) p[j] = -INFINITY;
                    mt = fmaxf(mt, p[j]);
                }
                if (pl.s && n < nh) {
    #pragma unroll
                    for (int t = 0; t < S::NT; ++t) {
                        float* to = pl.s + ((int64_t)it.row * a.hq + h0 + n) * pl.cap + it.p0 + i * S::TK + 16 * t + 4 * g;
                        *reinterpret_cast<v4f*>(to) = v4f{p[4 * t], p[4 * t + 1], p[4 * t + 2], p[4 * t + 3]};
                    }
                }
                mt = rows_max(mt);
                if (__any(mt > m)) {
                    const float f = pow2(m - (mt == -INFINITY ? 0.0f : mt));
                    m = mt;
                    l *= f;
    #pragma unroll
                    for (int x = 0; x < S::NU * S::UE; ++x) o[x] *= f;
                }
                const float base = m == -INFINITY ? 0.0f : m;
    #pragma unroll
                for (int j = 0; j < S::NJ; ++j) {
                    p[j] = pow2(p[j] - base);
                    l += p[j];
                }
                if (!was_full) {  // weights of 0 do not clear what is no number
    #pragma unroll
                    for (int j = 0; j < S::NJ; ++j)
                        if (of[16 * (j / 4) + 4 * g + j % 4] < 0)
    #pragma unroll
                            for (int u = 0; u < S::NU; ++u) vr[j][u] = v4i{0, 0, 0, 0};
                }
                if constexpr (S::F32) {
    #pragma unroll
                    for (int j = 0; j < S::NJ; ++j)
    #pragma unroll
                        for (int u = 0; u < S::NU; ++u)
    #pragma unroll
                            for (int e = 0; e < 4; ++e)
                                o[u * 4 + e] = __builtin_amdgcn_mfma_f32_16x16x4f32(__int_as_float(vr[j][u][e]), p[j],
                                                                                    o[u * 4 + e], 0, 0, 0);
                } else {
                    typename Split<DT>::V pp[3];
    #pragma unroll
                    for (int j = 0; j < 8; ++j) p[j] *= Split<DT>::P;
                    split8<DT>(p, pp);
    #pragma unroll
                    for (int u = 0; u < S::NU; ++u)
    #pragma unroll
                        for (int e = 0; e < S::UE; ++e) {
                            const unsigned sel = e % 2 ? 0x07060302u : 0x05040100u;
                            v4i col;
    #pragma unroll
                            for (int x = 0; x < 4; ++x)
                                col[x] = (int)__builtin_amdgcn_perm((unsigned)vr[2 * x + 1][u][e / 2],
                                                                    (unsigned)vr[2 * x][u][e / 2], sel);
                            const auto cv = __builtin_bit_cast(typename Split<DT>::V, col);
                            v4f& sum = o[u * S::UE + e];
                            if constexpr (Split<DT>::STEP == 1.0f) {
    #pragma unroll
                                for (int x = Split<DT>::N - 1; x >= 0; --x) sum = Split<DT>::mfma(cv, pp[x], sum);
                            } else {
                                v4f low = {0.0f, 0.0f, 0.0f, 0.0f};
    #pragma unroll
                                for (int x = Split<DT>::N - 1; x > 0; --x)
                                    low = Split<DT>::mfma(cv, pp[x], low) * (1.0f / Split<DT>::STEP);
                                sum = Split<DT>::mfma(cv, pp[0], sum + low);
                            }
                        }
                }
                if (i + kAttnWaves < ntiles) load_v(i + kAttnWaves);
            }
            l = rows_sum(l);
            if constexpr (!S::F32) {
    #pragma unroll
                for (int x = 0; x < S::NU * S::UE; ++x) o[x] *= 1.0f / Split<DT>::P;
            }
        }

        // The waves' sums, relative to the largest maximum
        bool bad = !fast;
        if (fast) {
            if (g == 0) {
                lds_ml[wave][0][n] = m;
                lds_ml[wave][1][n] = l;
            }
            __syncthreads();
            float mm = lds_ml[0][0][n];
    #pragma unroll
            for (int w = 1; w < kAttnWaves; ++w) mm = fmaxf(mm, lds_ml[w][0][n]);
            const float f = pow2(m - (mm == -INFINITY ? 0.0f : mm));
    #pragma unroll
            for (int u = 0; u < S::NU; ++u)
    #pragma unroll
                for (int r = 0; r < 4; ++r)
    #pragma unroll
                    for (int e = 0; e < S::UE; ++e) {
                        const int nom = 16 * S::UE * u + S::UE * (4 * g + r), d = min(nom, D - S::UE) + e;
                        if (d >= nom) lds_o[(wave * 16 + n) * kLdsRow + d] = o[u * S::UE + e][r] * f;
                    }
            __syncthreads();
            if (threadIdx.x < 16) {
                float lt = 0.0f;
                for (int w = 0; w < kAttnWaves; ++w)
                    lt += lds_ml[w][1][n] * pow2(lds_ml[w][0][n] - (mm == -INFINITY ? 0.0f : mm));
                lds_ml[0][0][n] = mm;
                lds_ml[0][1][n] = lt;
                bad = n < nh && !(mm < INFINITY && lt < INFINITY);
            }
            for (int x = threadIdx.x; x < nh * D; x += kAttnThreads) {
                const int h = x / D, d = x % D;
                float v = 0.0f;
    #pragma unroll
                for (int w = 0; w < kAttnWaves; ++w) v += lds_o[(w * 16 + h) * kLdsRow + d];
                lds_o[h * kLdsRow + d] = v;
                bad |= !(fabsf(v) < INFINITY);
            }
        }
        // Not all finite (or a tiny head): in plain operations.  (A segment of
        // nothing but holes has a maximum of -inf, sums of 0, and is done.)
        if (__syncthreads_or(bad)) attn_plain<DT>(a, pl, it, hk, h0, nh, scale2, lds_o, &lds_ml[0][0][0], kLdsRow);

        if (it.nc == 1) {
            float* to = a.out + it.row * a.ldo + (int64_t)h0 * D;
            for (int h = wave; h < nh; h += kAttnWaves) {
                const float lt = lds_ml[0][1][h];
                for (int d = lane; d < D; d += 64) to[h * D + d] = lt == 0.0f ? 0.0f : lds_o[h * kLdsRow + d] / lt;
            }
            if (threadIdx.x < nh) {
                const int64_t row_h = (int64_t)it.row * a.hq + h0 + n;
                const float mm = lds_ml[0][0][n], lt = lds_ml[0][1][n];
                if (a.lse) a.lse[row_h] = row_lse(mm, lt);
                if (pl.ml) {
                    pl.ml[2 * row_h] = mm;
                    pl.ml[2 * row_h + 1] = lt;
                }
            }
        } else {
            const int64_t item = ((int64_t)blockIdx.x + it.row) * pl.hy + blockIdx.y;
            for (int h = wave; h < nh; h += kAttnWaves)
                for (int d = 2 * lane; d < D; d += 128)
                    st2_device(pl.part_o + (item * 16 + h) * pl.dp + d, lds_o[h * kLdsRow + d],
                               d + 1 < D ? lds_o[h * kLdsRow + d + 1] : 0.0f);
            if (threadIdx.x < nh) st2_device(pl.part_ml + (item * 16 + n) * 2, lds_ml[0][0][n], lds_ml[0][1][n]);
            const int64_t slot = (int64_t)blockIdx.x + it.row, group = (slot - it.slot) / kJoinGroup;
            const int groups = (it.nc + kJoinGroup - 1) / kJoinGroup;
            const int64_t g0 = it.slot + group * kJoinGroup;
            const int in_group = (int)min((int64_t)kJoinGroup, it.slot + it.nc - g0);
            if (attention_count(pl.count + g0 * pl.hy + blockIdx.y, in_group, &lds_last)) {
                attention_join<DP>(a, pl, it.row, g0, 1, in_group, groups == 1, h0, nh, lds_o);
                if (groups > 1 &&
                    attention_count(pl.tops + (int64_t)it.row * pl.hy + blockIdx.y, groups, &lds_last))
                    attention_join<DP>(a, pl, it.row, it.slot, kJoinGroup, groups, true, h0, nh, lds_o);
            }
        }
        __syncthreads();
    }
}

// Adds the attention weights of a segment to the scores: one workgroup per
// (share, kv head), every query head of the group.
__device__ void attention_scores(const AttnArgs& a, const AttnPlan& pl, const AttnSeg& it, int hk) {
    const KvView& c = a.c;
    const int G = a.hq / c.hkv, sq = a.seq ? a.seq[it.row] : it.row;
    extern __shared__ float hm[];  // [G] maximum, [G] 1 / sum
    for (int h = threadIdx.x; h < G; h += kAttnThreads) {
        const float* ml = pl.ml + 2 * ((int64_t)it.row * a.hq + hk * G + h);
        hm[h] = ml[0] == -INFINITY ? 0.0f : ml[0];
        hm[G + h] = ml[1] == 0.0f ? 0.0f : 1.0f / ml[1];
    }
    __syncthreads();
    for (int p = it.p0 + threadIdx.x; p < it.p1; p += kAttnThreads) {
        const int pg = kv_page(c, sq, p);
        if (pg < 0) continue;
        float w = 0.0f;
        for (int h = 0; h < G; ++h)
            w += pow2(pl.s[((int64_t)it.row * a.hq + hk * G + h) * pl.cap + p] - hm[h]) * hm[G + h];
        atomicAdd(&c.score[((int64_t)pg * c.hkv + hk) * c.page + kv_slot(c, p)], w);
    }
}

__global__ __launch_bounds__(kAttnThreads) void attention_score_kernel(AttnArgs a, AttnPlan pl) {
    __shared__ int64_t lds_ends[kAttnPlanRows];
    const AttnLine line(a, pl, lds_ends);
    if ((int64_t)blockIdx.x >= line.x) return;
    int64_t at = line.begin(blockIdx.x);
    const int64_t to = line.begin(blockIdx.x + 1);
    for (int r = line.row_at(at); at < to; ++r) {
        int64_t row_end;
        const AttnSeg it = line.segment(r, at, to, &row_end);
        at = row_end;
        attention_scores(a, pl, it, blockIdx.y);
        __syncthreads();
    }
}

namespace {

// Workgroups of attention_kernel per compute unit that the work is split for:
// as many as it holds by registers with a 16-bit cache.  The f32 kernels take
// fewer and one more of each would fit up to 128: measured slower (9 rows, 32
// heads of 100: 86 us with two, 95 with three; 64 rows, 8 kv heads of 128, 182 and
// 190; of 64, 100 with three and 102 with four).
int resident(int D) { return D > 128 ? 1 : (D > 64 ? 2 : 3); }

AttnPlan make_plan(const AttnArgs& a, int cus) {
    AttnPlan pl;
    const int G = a.hq / a.c.hkv;
    pl.part_o = pl.part_ml = pl.s = pl.ml = nullptr;
    pl.count = pl.tops = nullptr;
    pl.dp = (a.c.D + 1) / 2 * 2;
    pl.tiles = (G + 15) / 16;
    pl.hy = a.c.hkv * pl.tiles;
    const int64_t cap = (int64_t)a.c.max_pages * a.c.page;
    pl.cap = (cap + 31) / 32 * 32;
    pl.per_row = a.call_rows > kAttnPlanRows;
    const int64_t steps = a.R * std::max<int64_t>(1, (cap + kAttnStep - 1) / kAttnStep);
    pl.shares = (int)std::min(steps, std::max<int64_t>(1, (int64_t)resident(a.c.D) * cus / pl.hy));
    pl.shares = std::min(pl.shares, 64 * kJoinGroup);  // (as many as two levels join)
    if (pl.per_row) pl.shares = (int)a.R;
    return pl;
}

// Whether a row may be in more than one segment.
bool splits(const AttnArgs& a, const AttnPlan& pl) {
    return !pl.per_row && (int64_t)a.c.max_pages * a.c.page > kAttnStep;
}

template <int DT>
hipError_t launch_attention(const AttnArgs& a, const AttnPlan& pl, hipStream_t s) {
    const dim3 grid((unsigned)pl.shares, (unsigned)pl.hy), block(kAttnThreads);
    const float scale2 = (float)((double)a.scale * 1.4426950408889634);
    if (a.c.D <= 64)
        attention_kernel<DT, 64><<<grid, block, 0, s>>>(a, pl, scale2);
    else if (a.c.D <= 128)
        attention_kernel<DT, 128><<<grid, block, 0, s>>>(a, pl, scale2);
    else
        attention_kernel<DT, 256><<<grid, block, 0, s>>>(a, pl, scale2);
    return hipGetLastError();
}

// Bytes of the plan's arrays in one workspace.
size_t place(const AttnArgs& a, AttnPlan* pl, char* base) {
    size_t at = 0;
    auto take = [&](size_t floats) {
        float* p = reinterpret_cast<float*>(base + at);
        at += (floats * 4 + 255) / 256 * 256;
        return p;
    };
    const size_t slots = (size_t)pl->shares + (size_t)a.R;
    if (splits(a, *pl)) {
        pl->part_ml = take(slots * pl->hy * 32);
        pl->part_o = take(slots * pl->hy * 16 * pl->dp);
    }
    if (a.accumulate) {
        pl->ml = take((size_t)a.R * a.hq * 2);
        pl->s = take((size_t)a.R * a.hq * pl->cap);
    }
    return at;
}

}  // namespace

size_t attention_workspace(const AttnArgs& a, int cus, size_t* counters) {
    AttnPlan pl = make_plan(a, cus);
    *counters = splits(a, pl) ? ((size_t)pl.shares + 2 * (size_t)a.R) * pl.hy * sizeof(unsigned) : 0;
    return place(a, &pl, nullptr);
}

hipError_t launch_paged_attention(int dtype, const AttnArgs& a, int cus, void* ws, void* counters, hipStream_t s) {
    AttnPlan pl = make_plan(a, cus);
    (void)place(a, &pl, static_cast<char*>(ws));
    pl.count = static_cast<unsigned*>(counters);
    pl.tops = pl.count + ((size_t)pl.shares + (size_t)a.R) * pl.hy;
    hipError_t e;
    switch (dtype) {
        case XT_F32: e = launch_attention<XT_F32>(a, pl, s); break;
        case XT_F16: e = launch_attention<XT_F16>(a, pl, s); break;
        default: e = launch_attention<XT_BF16>(a, pl, s); break;
    }
    if (e != hipSuccess || !a.accumulate) return e;
    const size_t lds = 2 * sizeof(float) * (size_t)(a.hq / a.c.hkv);
    attention_score_kernel<<<dim3((unsigned)pl.shares, (unsigned)a.c.hkv), kAttnThreads, lds, s>>>(a, pl);
    return hipGetLastError();
}

}  // namespace xt
