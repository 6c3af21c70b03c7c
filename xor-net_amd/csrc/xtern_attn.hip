// The paged key-value cache's append (rotary embedding, rounding, scatter)
// and the attention of one token per row over it.
#include <algorithm>

#include "xtern_cache.h"
#include "xtern_device.h"

namespace xt {

// ---------------------------------------------------------------------------
// Append
// ---------------------------------------------------------------------------
// With h = rot / 2, element i < h of a rotated head becomes
//   x[i] cos - x[i + h] sin,   element i + h   x[i + h] cos + x[i] sin
// (cos, sin: row `pos`, column i of the tables); elements from rot on, and
// values, are copied.  One thread per pair (i, i + h) or per copied element.
template <int DT>
__global__ __launch_bounds__(256) void kv_append_kernel(AppendArgs a) {
    typedef Elem<DT> E;
    const int64_t r = blockIdx.x;
    const KvView& c = a.c;
    const int slot = a.slots[r];
    const int sq = a.seq ? a.seq[r] : (int)r;
    if (slot < 0 || slot >= (int64_t)c.max_pages * c.page || (unsigned)sq >= (unsigned)c.nseq) return;
    const int pg = kv_page(c, sq, slot);
    if (pg < 0) return;
    const int pos = a.cos ? a.pos[r] : 0;
    if (a.cos && (pos < 0 || pos >= a.rope_rows)) return;
    const int half = a.cos ? a.rot / 2 : 0, rest = c.D - 2 * half;
    const int per = half + rest;  // threads' work items of one head
    const int hq = a.q ? a.hq : 0;
    const int nq = hq * per, nk = c.hkv * per, nv = c.hkv * c.D;
    typename E::T* kc = static_cast<typename E::T*>(c.k);
    typename E::T* vc = static_cast<typename E::T*>(c.v);
    for (int i = threadIdx.x; i < nq + nk + nv; i += blockDim.x) {
        if (i >= nq + nk) {
            const int j = i - nq - nk, h = j / c.D, d = j % c.D;
            vc[kv_offset(c, pg, slot, h) + d] = E::put(a.v[r * a.ldv + j]);
            if (c.score && d == 0) c.score[((int64_t)pg * c.hkv + h) * c.page + slot % c.page] = 0.0f;
            continue;
        }
        const bool isq = i < nq;
        const int j = isq ? i : i - nq, h = j / per, e = j % per;
        const float* x = isq ? a.q + r * a.ldq + (int64_t)h * c.D : a.k + r * a.ldk + (int64_t)h * c.D;
        float y0, y1 = 0.0f;
        int d0 = e, d1 = -1;
        if (e < half) {
            d1 = e + half;
            const float cs = a.cos[(int64_t)pos * half + e], sn = a.sin[(int64_t)pos * half + e];
            const float x0 = x[d0], x1 = x[d1];
            y0 = x0 * cs - x1 * sn;
            y1 = x1 * cs + x0 * sn;
        } else {
            d0 = e + half;
            y0 = x[d0];
        }
        if (isq) {
            float* o = a.qo + r * a.ldqo + (int64_t)h * c.D;
            o[d0] = y0;
            if (d1 >= 0) o[d1] = y1;
        } else {
            typename E::T* o = kc + kv_offset(c, pg, slot, h);
            o[d0] = E::put(y0);
            if (d1 >= 0) o[d1] = E::put(y1);
        }
    }
}

hipError_t launch_kv_append(int dtype, const AppendArgs& a, hipStream_t s) {
    const dim3 grid((unsigned)a.R), block(256);
    switch (dtype) {
        case XT_F32: kv_append_kernel<XT_F32><<<grid, block, 0, s>>>(a); break;
        case XT_F16: kv_append_kernel<XT_F16><<<grid, block, 0, s>>>(a); break;
        default: kv_append_kernel<XT_BF16><<<grid, block, 0, s>>>(a); break;
    }
    return hipGetLastError();
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
// 16-bit caches: q and p in f32 are split into bf16 (three pieces) or f16 (two,
// scaled by a power of two against its short range), whose products with k, v
// the 16-bit MFMA adds up exactly in f32: the matrix cores have that to spare
// (24 instructions of 16 cycles per 32 positions and piece-of-three against
// 6700 cycles of HBM time).  f32 caches take the f32 MFMA.

typedef float v4f __attribute__((ext_vector_type(4)));
typedef int v2i __attribute__((ext_vector_type(2)));
typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
// (rows may start at any element: the hardware loads unaligned vectors)
typedef v4i v4iu __attribute__((aligned(2)));
typedef v2i v2iu __attribute__((aligned(2)));

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
// More than kAttnPlanRows rows: one workgroup per row.
struct AttnPlan {
    float* part_o;   // [slots][hy][16][D], unnormalised, relative to the segment's maximum
    float* part_ml;  // [slots][hy][2][16]: maximum (base 2), sum
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

// The line as every wave of the workgroup sees it: 64 rows, a lane each, in
// registers (no barrier), or the rows' ends in LDS.
struct AttnLine {
    const AttnArgs& a;
    const AttnPlan& pl;
    int len, upto;       // the lane's row (R <= 64)
    int64_t* ends;       // LDS, [R] (R > 64)
    int64_t total;       // steps
    int x;               // shares that the line is cut into

    __device__ AttnLine(const AttnArgs& a_, const AttnPlan& pl_, int64_t* lds) : a(a_), pl(pl_), ends(lds) {
        if (pl.per_row) {
            total = x = (int)a.R;
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
        x = (int)min((int64_t)pl.shares, total);
    }
    // First step of share b; the share that holds a step.
    __device__ int64_t begin(int b) const { return (int64_t)b * total / x; }
    __device__ int share_of(int64_t step) const { return (int)(((step + 1) * x - 1) / total); }
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

template <int DT> struct Split;  // pieces of an f32 operand
template <> struct Split<XT_BF16> {
    typedef v8bf V;
    static constexpr int N = 3;
    static constexpr float P = 1.0f;  // scale of the probabilities
    static __device__ __forceinline__ v4f mfma(V a, V b, v4f c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
    }
};
template <> struct Split<XT_F16> {
    typedef v8h V;
    static constexpr int N = 2;
    // p <= 1: 2^14 p fits f16, and what its two pieces leave is below 2^-25 of
    // the largest
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
            r[i] -= (float)p;
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
    static constexpr int QV = F32 ? KS : KS * Split<F32 ? (int)XT_BF16 : DT>::N;  // query registers (16 bytes)
};

// One chunk [p0, p1) of a row for the heads h0 .. h0 + nh - 1, in plain f32
// operations: what the matrix cores' split operands cannot give (infinities
// and NaN among the inputs, sums past f32's range in a piece) and head sizes
// below one load.  256 positions at a time, one head after the other.  Writes
// the sums as attention_item does.
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

template <int DT, int DP>
__global__ __launch_bounds__(kAttnThreads, DP == 256 ? 1 : (DP == 128 || DT != XT_F32 ? 2 : 3)) void attention_kernel(AttnArgs a, AttnPlan pl,
                                                                                   float scale2) {
    typedef AttnShape<DT, DP> S;
    typedef Elem<DT> E;
    typedef typename E::T T;
    const KvView& c = a.c;
    constexpr int kLdsRow = DP + 4;  // floats; the pad keeps heads apart in the banks
    __shared__ float lds_o[kAttnWaves * 16 * kLdsRow];
    __shared__ float lds_ml[kAttnWaves][2][16];
    __shared__ int64_t lds_off[kAttnWaves][2][32];
    __shared__ int64_t lds_ends[kAttnPlanRows];
    const int hk = blockIdx.y / pl.tiles, G = a.hq / c.hkv;
    const int h0 = hk * G + (blockIdx.y % pl.tiles) * 16, nh = min(16, hk * G + G - h0);
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
    const int D = c.D;
    const bool fast = D >= S::KU;
    const AttnLine line(a, pl, lds_ends);
    if ((int)blockIdx.x >= line.x) return;
    int64_t at = line.begin(blockIdx.x);
    const int64_t to_step = line.begin(blockIdx.x + 1);
    for (int r = line.row_at(at); at < to_step; ++r) {
        int64_t row_end;
        const AttnSeg it = line.segment(r, at, to_step, &row_end);
        at = row_end;
        const int sq = a.seq ? a.seq[r] : r;
        const int ntiles = it.p1 > it.p0 ? (it.p1 - it.p0 + S::TK - 1) / S::TK : 0;

        float m = -INFINITY, l = 0.0f, qs = scale2;
        v4f o[S::NU * S::UE];
    #pragma unroll
        for (int i = 0; i < S::NU * S::UE; ++i) o[i] = v4f{0.0f, 0.0f, 0.0f, 0.0f};

        if (fast && wave < ntiles) {
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
                return p < it.p1 ? c.table[(int64_t)sq * c.ldt + p / c.page] : -1;
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
            auto load_v = [&](int i) {
                const int64_t* of = lds_off[wave][(i / kAttnWaves) & 1];
    #pragma unroll
                for (int j = 0; j < S::NJ; ++j) {
                    const T* row = vc + max(of[16 * (j / 4) + 4 * g + j % 4], (int64_t)0);
    #pragma unroll
                    for (int u = 0; u < S::NU; ++u) {
                        if constexpr (S::UE * S::ES == 16) {
                            vr[j][u] = *reinterpret_cast<const v4iu*>(row + vd[u]);
                        } else {
                            const v2i x = *reinterpret_cast<const v2iu*>(row + vd[u]);
                            vr[j][u] = v4i{x[0], x[1], 0, 0};
                        }
                    }
                }
            };

            int next_e = entry(wave);
            const int after_e = entry(wave + kAttnWaves);
            // the lane's pieces of the query rows: head h0 + n, elements from
            // min(KU (4 s + g), D - KU); where pieces overlap (D no multiple of
            // KU, or past D) the earlier one counts, the later one holds zeros
            const float* q = a.q + it.row * a.ldq + (int64_t)(h0 + (n < nh ? n : 0)) * D;
            float qf[S::KS * S::KU];
    #pragma unroll
            for (int i = 0; i < S::KS * S::KU; ++i) qf[i] = q[kd[i / S::KU] + i % S::KU];
            bool full = offsets(wave, next_e);
            next_e = after_e;
            load_k(wave);
            load_v(wave);
            // (the queries' arithmetic while the first tile is on its way)
    #pragma unroll
            for (int i = 0; i < S::KS * S::KU; ++i)
                if (n >= nh || kd[i / S::KU] + i % S::KU < S::KU * (4 * (i / S::KU) + g)) qf[i] = 0.0f;
            typename Split<S::F32 ? (int)XT_BF16 : DT>::V qp[S::F32 ? 1 : S::KS][3];
            if constexpr (!S::F32) {
                if constexpr (DT == XT_F16) {
                    // the row's largest element at 2^14 .. 2^15: f16's two pieces
                    // then hold 22 bits of every element, or 2^-39 of the largest
                    float mx = 0.0f;
    #pragma unroll
                    for (int i = 0; i < S::KS * S::KU; ++i) mx = fmaxf(mx, fabsf(qf[i]));
                    mx = rows_max(mx);
                    int e = 0;
                    if (mx > 0.0f && mx < INFINITY) {
                        (void)frexpf(mx, &e);
                        e = max(-100, min(100, 15 - e));
                    }
                    const float up = ldexpf(1.0f, e);
                    qs = scale2 * ldexpf(1.0f, -e);
    #pragma unroll
                    for (int i = 0; i < S::KS * S::KU; ++i) qf[i] *= up;
                }
    #pragma unroll
                for (int s = 0; s < S::KS; ++s) split8<DT>(&qf[s * S::KU], qp[s]);
            }
            for (int i = wave; i < ntiles; i += kAttnWaves) {
                // S of the tile
                v4f sc[S::NT];
    #pragma unroll
                for (int t = 0; t < S::NT; ++t) {
                    sc[t] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
                    if constexpr (S::F32) {
    #pragma unroll
                        for (int s = 0; s < S::KS; ++s)
    #pragma unroll
                            for (int x = 0; x < 4; ++x)
                                sc[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(__int_as_float(kr[t][s][x]), qf[s * 4 + x],
                                                                             sc[t], 0, 0, 0);
                    } else {
    #pragma unroll
                        for (int s = 0; s < S::KS; ++s)
    #pragma unroll
                            for (int x = Split<DT>::N - 1; x >= 0; --x)
                                sc[t] = Split<DT>::mfma(__builtin_bit_cast(typename Split<DT>::V, kr[t][s]), qp[s][x],
                                                        sc[t]);
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
    #pragma unroll
                            for (int x = Split<DT>::N - 1; x >= 0; --x)
                                o[u * S::UE + e] = Split<DT>::mfma(__builtin_bit_cast(typename Split<DT>::V, col), pp[x],
                                                                   o[u * S::UE + e]);
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
                bad = n < nh && !(fabsf(mm) < INFINITY && lt < INFINITY) && it.p1 > it.p0;
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
        // Not all finite (or a tiny head): in plain operations.  (A row of holes
        // has a maximum of -inf and comes here too.)
        if (__syncthreads_or(bad)) attn_plain<DT>(a, pl, it, hk, h0, nh, scale2, lds_o, &lds_ml[0][0][0], kLdsRow);

        const bool whole = it.nc == 1;
        const int64_t item = ((int64_t)blockIdx.x + it.row) * pl.hy + blockIdx.y;
        float* to = whole ? a.out + it.row * a.ldo + (int64_t)h0 * D : pl.part_o + item * 16 * D;
        for (int x = threadIdx.x; x < nh * D; x += kAttnThreads) {
            const int h = x / D, d = x % D;
            const float v = lds_o[h * kLdsRow + d], lt = lds_ml[0][1][h];
            to[x] = !whole ? v : (lt == 0.0f ? 0.0f : v / lt);
        }
        if (threadIdx.x < nh) {
            const float mm = lds_ml[0][0][n], lt = lds_ml[0][1][n];
            if (whole && a.lse)
                a.lse[(int64_t)it.row * a.hq + h0 + n] = lt == 0.0f ? -INFINITY : (mm + log2f(lt)) * 0.69314718056f;
            if (pl.part_ml) {
                pl.part_ml[item * 32 + n] = mm;
                pl.part_ml[item * 32 + 16 + n] = lt;
            }
        }
        __syncthreads();
    }
}

// Joins the segments of a row: one workgroup per (row, query head).  The
// factors of 256 segments at a time go to LDS, then every thread adds up four
// columns of every eighth (or fourth) segment, eight loads in flight.
__device__ void attention_join(const AttnArgs& a, const AttnPlan& pl, const AttnLine& line, int row) {
    int64_t row_end;
    const AttnSeg it = line.segment(row, 0, INT64_MAX, &row_end);
    if (it.nc == 1) return;
    const int G = a.hq / a.c.hkv, h = blockIdx.y, hk = h / G, tile = (h % G) / 16, n = (h % G) % 16;
    const int D = a.c.D, t = threadIdx.x, wave = t >> 6;
    __shared__ float sf[kAttnThreads];
    __shared__ float so[kAttnThreads * 4];
    __shared__ float sm[2][kAttnWaves];
    const int64_t first = (int64_t)it.slot * pl.hy + hk * pl.tiles + tile;
    const int64_t stride = (int64_t)pl.hy * 16 * D;  // of part_o, chunk to chunk
    const float* po = pl.part_o + (first * 16 + n) * D;
    const int cols = D <= 128 ? 32 : 64, groups = kAttnThreads / cols;
    const int c4 = (t % cols) * 4, grp = t / cols;
    float m = -INFINITY, l = 0.0f, v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int c0 = 0; c0 < it.nc; c0 += kAttnThreads) {
        const int cnt = min(kAttnThreads, it.nc - c0);
        const float* ml = pl.part_ml + (first + (int64_t)(c0 + min(t, cnt - 1)) * pl.hy) * 32 + n;
        const float mc = t < cnt ? ml[0] : -INFINITY, lc = t < cnt ? ml[16] : 0.0f;
        const float mw = wave_max(mc);
        __syncthreads();  // (the last round's factors are used up)
        if ((t & 63) == 0) sm[0][wave] = mw;
        __syncthreads();
        const float mn = fmaxf(m, fmaxf(fmaxf(sm[0][0], sm[0][1]), fmaxf(sm[0][2], sm[0][3])));
        const float base = mn == -INFINITY ? 0.0f : mn;
        const float f = pow2(m - base), fc = pow2(mc - base);
        sf[t] = fc;
        const float lw = wave_sum(lc * fc);
        if ((t & 63) == 0) sm[1][wave] = lw;
        m = mn;
        __syncthreads();
        l = l * f + ((sm[1][0] + sm[1][1]) + (sm[1][2] + sm[1][3]));
#pragma unroll
        for (int x = 0; x < 4; ++x) v[x] *= f;
        for (int c = grp; c < cnt; c += 8 * groups) {
            float ld[8][4], w[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                const int cu = c + u * groups;
                w[u] = cu < cnt ? sf[cu] : 0.0f;
                const float* o = po + (int64_t)(c0 + min(cu, cnt - 1)) * stride;
#pragma unroll
                for (int x = 0; x < 4; ++x) ld[u][x] = o[min(c4 + x, D - 1)];
            }
#pragma unroll
            for (int u = 0; u < 8; ++u)
#pragma unroll
                for (int x = 0; x < 4; ++x) v[x] += c + u * groups < cnt ? w[u] * ld[u][x] : 0.0f;
        }
    }
    // [group][4 cols]
    __syncthreads();
#pragma unroll
    for (int x = 0; x < 4; ++x) so[grp * 4 * cols + c4 + x] = v[x];
    __syncthreads();
    if (t < D) {
        float s = 0.0f;
        for (int gI = 0; gI < groups; ++gI) s += so[gI * 4 * cols + t];
        a.out[it.row * a.ldo + (int64_t)h * D + t] = l == 0.0f ? 0.0f : s / l;
    }
    if (t == 0 && a.lse)
        a.lse[(int64_t)it.row * a.hq + h] = l == 0.0f ? -INFINITY : (m + log2f(l)) * 0.69314718056f;
}

// Adds the attention weights of a segment to the scores: one workgroup per
// (share, kv head), every query head of the group.
__device__ void attention_scores(const AttnArgs& a, const AttnPlan& pl, const AttnSeg& it, int hk) {
    const KvView& c = a.c;
    const int G = a.hq / c.hkv, sq = a.seq ? a.seq[it.row] : it.row;
    extern __shared__ float hm[];  // [G] maximum, [G] 1 / sum
    // a wave per head, a lane per chunk
    for (int h = threadIdx.x >> 6; h < G; h += kAttnWaves) {
        const int64_t first = (int64_t)it.slot * pl.hy + hk * pl.tiles + h / 16;
        float m = -INFINITY, l = 0.0f;
        for (int x = threadIdx.x & 63; x < it.nc; x += 64) {
            const float* ml = pl.part_ml + (first + (int64_t)x * pl.hy) * 32 + h % 16;
            const float mn = fmaxf(m, ml[0]), base = mn == -INFINITY ? 0.0f : mn;
            l = l * pow2(m - base) + ml[16] * pow2(ml[0] - base);
            m = mn;
        }
        const float mw = wave_max(m), base = mw == -INFINITY ? 0.0f : mw;
        l = wave_sum(l * pow2(m - base));
        if ((threadIdx.x & 63) == 0) {
            hm[h] = base;
            hm[G + h] = l == 0.0f ? 0.0f : 1.0f / l;
        }
    }
    __syncthreads();
    for (int p = it.p0 + threadIdx.x; p < it.p1; p += kAttnThreads) {
        const int pg = kv_page(c, sq, p);
        if (pg < 0) continue;
        float w = 0.0f;
        for (int h = 0; h < G; ++h)
            w += pow2(pl.s[((int64_t)it.row * a.hq + hk * G + h) * pl.cap + p] - hm[h]) * hm[G + h];
        atomicAdd(&c.score[((int64_t)pg * c.hkv + hk) * c.page + p % c.page], w);
    }
}

// What follows the attention kernel: workgroups (x, y < hq) join row x of
// query head y, workgroups (x, hq + kv head) add share x's weights.
__global__ __launch_bounds__(kAttnThreads) void attention_finish_kernel(AttnArgs a, AttnPlan pl) {
    __shared__ int64_t lds_ends[kAttnPlanRows];
    const AttnLine line(a, pl, lds_ends);
    if ((int)blockIdx.y < a.hq) {
        if (blockIdx.x < a.R) attention_join(a, pl, line, blockIdx.x);
        return;
    }
    if ((int64_t)blockIdx.x >= line.x) return;
    int64_t at = line.begin(blockIdx.x);
    const int64_t to = line.begin(blockIdx.x + 1);
    for (int r = line.row_at(at); at < to; ++r) {
        int64_t row_end;
        const AttnSeg it = line.segment(r, at, to, &row_end);
        at = row_end;
        attention_scores(a, pl, it, (int)blockIdx.y - a.hq);
        __syncthreads();
    }
}

namespace {

// Workgroups of attention_kernel that a compute unit holds, by registers.
int resident(int dtype, int D) { return D > 128 ? 1 : (D > 64 || dtype != XT_F32 ? 2 : 3); }

AttnPlan make_plan(int dtype, const AttnArgs& a, int cus) {
    AttnPlan pl;
    const int G = a.hq / a.c.hkv;
    pl.part_o = pl.part_ml = pl.s = nullptr;
    pl.tiles = (G + 15) / 16;
    pl.hy = a.c.hkv * pl.tiles;
    const int64_t cap = (int64_t)a.c.max_pages * a.c.page;
    pl.cap = (cap + 31) / 32 * 32;
    pl.per_row = a.R > kAttnPlanRows;
    const int64_t steps = a.R * std::max<int64_t>(1, (cap + kAttnStep - 1) / kAttnStep);
    pl.shares = (int)std::min(steps, std::max<int64_t>(1, (int64_t)resident(dtype, a.c.D) * cus / pl.hy));
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
    pl->part_ml = take(slots * pl->hy * 32);
    if (splits(a, *pl)) pl->part_o = take(slots * pl->hy * 16 * a.c.D);
    if (a.accumulate) pl->s = take((size_t)a.R * a.hq * pl->cap);
    return at;
}

}  // namespace

size_t attention_workspace(int dtype, const AttnArgs& a, int cus) {
    AttnPlan pl = make_plan(dtype, a, cus);
    return splits(a, pl) || a.accumulate ? place(a, &pl, nullptr) : 0;
}

hipError_t launch_paged_attention(int dtype, const AttnArgs& a, int cus, void* ws, hipStream_t s) {
    AttnPlan pl = make_plan(dtype, a, cus);
    if (ws) (void)place(a, &pl, static_cast<char*>(ws));
    hipError_t e;
    switch (dtype) {
        case XT_F32: e = launch_attention<XT_F32>(a, pl, s); break;
        case XT_F16: e = launch_attention<XT_F16>(a, pl, s); break;
        default: e = launch_attention<XT_BF16>(a, pl, s); break;
    }
    if (e != hipSuccess || !ws) return e;
    // (rows are not joined where none is split)
    const dim3 grid((unsigned)std::max<int64_t>(a.R, a.accumulate ? pl.shares : 0),
                    (unsigned)(a.hq + (a.accumulate ? a.c.hkv : 0)));
    const size_t lds = a.accumulate ? 2 * sizeof(float) * (size_t)(a.hq / a.c.hkv) : 0;
    attention_finish_kernel<<<grid, kAttnThreads, lds, s>>>(a, pl);
    return hipGetLastError();
}

}  // namespace xt
