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
constexpr int kAttnStep = 128;     // positions per chunk: multiples of this
constexpr int kAttnPlanRows = 1024;  // rows whose work is split by its total

// Split of the rows into work items of consecutive positions.
struct AttnPlan {
    float* part_o;   // [items][hy][16][D], unnormalised, relative to the item's maximum
    float* part_ml;  // [items][hy][2][16]: maximum (base 2), sum
    float* s;        // accumulate: S in base 2, [R][hq][cap]
    int64_t cap;     // positions of a row of s, a multiple of 32
    int hy;          // workgroups per item: kv heads x tiles of 16 query heads
    int tiles;       // of 16 query heads per kv head
    int target;      // items wanted
    int fixed;       // 0, or that many items per row (more than kAttnPlanRows rows)
};

struct AttnItem {
    int row, n, chunk, nc, p0, p1, base;  // base: the row's first item
};

__device__ __forceinline__ int attn_len(const AttnArgs& a, int64_t r) {
    const int sq = a.seq ? a.seq[r] : (int)r;
    return (unsigned)sq < (unsigned)a.c.nseq ? kv_length(a.c, a.lengths[r]) : 0;
}

// Positions per chunk for v wanted: whole steps, one at least; 2^30 holds
// every row (and the sum of two such lengths is an int).
__device__ __forceinline__ int chunk_len(int64_t v) {
    const int64_t len = (v + kAttnStep - 1) / kAttnStep * kAttnStep;
    return (int)max((int64_t)kAttnStep, min(len, (int64_t)1 << 30));
}

// Sum over the workgroup of v, and the sum over the threads before this one.
__device__ __forceinline__ int64_t wg_scan(int64_t v, int64_t* before, int64_t* sm) {
    int64_t x = v;
    for (int o = 1; o < 64; o <<= 1) {
        const int64_t y = __shfl_up(x, o);
        if ((int)(threadIdx.x & 63) >= o) x += y;
    }
    __syncthreads();
    if ((threadIdx.x & 63) == 63) sm[threadIdx.x >> 6] = x;
    __syncthreads();
    int64_t sum = 0, b = x - v;
    for (int w = 0; w < kAttnWaves; ++w) {
        if (w < (int)(threadIdx.x >> 6)) b += sm[w];
        sum += sm[w];
    }
    *before = b;
    return sum;
}

// The item `it` (of_row false) or the items of row `it` (true); false: none.
// Every thread of the workgroup calls it.  Up to kAttnPlanRows rows the chunk
// length is the same for all: the total of the lengths over the items wanted,
// so that short and long rows of a batch give work of one size.
__device__ bool attn_plan(const AttnArgs& a, const AttnPlan& pl, int it, bool of_row, AttnItem* out) {
    __shared__ int64_t sm[kAttnWaves];
    __shared__ AttnItem found;
    AttnItem f;
    if (pl.fixed) {
        f.row = of_row ? it : it / pl.fixed;
        f.chunk = of_row ? 0 : it % pl.fixed;
        f.base = f.row * pl.fixed;
        f.n = attn_len(a, f.row);
        const int len = chunk_len(((int64_t)f.n + pl.fixed - 1) / pl.fixed);
        f.nc = max(1, (f.n + len - 1) / len);
        if (f.chunk >= f.nc) return false;
        f.p0 = f.chunk * len;
        f.p1 = min(f.p0 + len, f.n);
        *out = f;
        return true;
    }
    constexpr int kPer = kAttnPlanRows / kAttnThreads;
    int len[kPer];
    int64_t sum = 0, before;
    const int per = ((int)a.R + kAttnThreads - 1) / kAttnThreads, r0 = threadIdx.x * per;
    for (int i = 0; i < kPer; ++i) {
        len[i] = i < per && r0 + i < a.R ? attn_len(a, r0 + i) : -1;
        sum += max(len[i], 0);
    }
    sum = wg_scan(sum, &before, sm);
    const int step = chunk_len((sum + pl.target - 1) / pl.target);
    int64_t mine = 0;
    for (int i = 0; i < kPer; ++i)
        if (len[i] >= 0) mine += max(1, (len[i] + step - 1) / step);
    const int64_t total = wg_scan(mine, &before, sm);
    if (!of_row && it >= total) return false;
    for (int i = 0; i < kPer; ++i) {
        if (len[i] < 0) continue;
        const int nc = max(1, (len[i] + step - 1) / step);
        if (of_row ? r0 + i == it : (it >= before && it < before + nc)) {
            f.row = r0 + i;
            f.n = len[i];
            f.base = (int)before;
            f.nc = nc;
            f.chunk = of_row ? 0 : it - (int)before;
            f.p0 = f.chunk * step;
            f.p1 = min(f.p0 + step, len[i]);
            found = f;
        }
        before += nc;
    }
    __syncthreads();
    *out = found;
    return true;
}

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

// 2^(v - m) with everything that is not there, or -inf, as 0.
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
__device__ void attn_plain(const AttnArgs& a, const AttnPlan& pl, const AttnItem& it, int hk, int h0, int nh,
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
__global__ __launch_bounds__(kAttnThreads, DP == 256 ? 1 : 2) void attention_kernel(AttnArgs a, AttnPlan pl,
                                                                                   float scale2) {
    typedef AttnShape<DT, DP> S;
    typedef Elem<DT> E;
    typedef typename E::T T;
    const KvView& c = a.c;
    constexpr int kLdsRow = DP + 4;  // floats; the pad keeps heads apart in the banks
    __shared__ float lds_o[kAttnWaves * 16 * kLdsRow];
    __shared__ float lds_ml[kAttnWaves][2][16];
    __shared__ int64_t lds_off[kAttnWaves][2][32];
    AttnItem it;
    if (!attn_plan(a, pl, blockIdx.x, false, &it)) return;
    const int hk = blockIdx.y / pl.tiles, G = a.hq / c.hkv;
    const int h0 = hk * G + (blockIdx.y % pl.tiles) * 16, nh = min(16, hk * G + G - h0);
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
    const int D = c.D, sq = a.seq ? a.seq[it.row] : it.row;
    const int ntiles = it.p1 > it.p0 ? (it.p1 - it.p0 + S::TK - 1) / S::TK : 0;
    const bool fast = D >= S::KU;

    float m = -INFINITY, l = 0.0f, qs = scale2;
    v4f o[S::NU * S::UE];
#pragma unroll
    for (int i = 0; i < S::NU * S::UE; ++i) o[i] = v4f{0.0f, 0.0f, 0.0f, 0.0f};

    if (fast && wave < ntiles) {
        // the lane's pieces of the query rows: head h0 + n, elements from
        // min(KU (4 s + g), D - KU); where pieces overlap (D no multiple of
        // KU, or past D) the earlier one counts, the later one holds zeros
        const float* q = a.q + it.row * a.ldq + (int64_t)(h0 + (n < nh ? n : 0)) * D;
        auto q_at = [&](int s, int i) {
            const int nom = S::KU * (4 * s + g), d = min(nom, D - S::KU) + i;
            return n < nh && d >= nom ? q[d] : 0.0f;
        };
        float qf[S::F32 ? S::KS * 4 : 1];
        typename Split<S::F32 ? (int)XT_BF16 : DT>::V qp[S::F32 ? 1 : S::KS][3];
        if constexpr (S::F32) {
#pragma unroll
            for (int i = 0; i < S::KS * 4; ++i) qf[i] = q_at(i / 4, i % 4);
        } else {
            float up = 1.0f;
            if constexpr (DT == XT_F16) {
                // the row's largest element at 2^14 .. 2^15 (f16's two pieces
                // then hold 22 bits of every element down to 2^-28 of it)
                float mx = 0.0f;
                for (int s = 0; s < S::KS; ++s)
                    for (int i = 0; i < S::KU; ++i) mx = fmaxf(mx, fabsf(q_at(s, i)));
                mx = rows_max(mx);
                int e = 0;
                if (mx > 0.0f && mx < INFINITY) (void)frexpf(mx, &e);
                e = max(-100, min(100, 15 - e));
                if (mx > 0.0f) {
                    up = ldexpf(1.0f, e);
                    qs = scale2 * ldexpf(1.0f, -e);
                }
            }
#pragma unroll
            for (int s = 0; s < S::KS; ++s) {
                float x[8];
                for (int i = 0; i < 8; ++i) x[i] = q_at(s, i) * up;
                split8<DT>(x, qp[s]);
            }
        }

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

        bool full = offsets(wave, entry(wave));
        load_k(wave);
        load_v(wave);
        int next_e = entry(wave + kAttnWaves);
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
    const int64_t item = (int64_t)(it.base + it.chunk) * pl.hy + blockIdx.y;
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
}

// Joins the chunks of a row.  One workgroup per (row, query head): a quarter
// of the chunks per wave, four columns per lane.
__global__ __launch_bounds__(kAttnThreads) void attention_join_kernel(AttnArgs a, AttnPlan pl) {
    AttnItem it;
    attn_plan(a, pl, blockIdx.x, true, &it);
    if (it.nc == 1) return;
    const int G = a.hq / a.c.hkv, h = blockIdx.y, hk = h / G, tile = (h % G) / 16, n = (h % G) % 16;
    const int D = a.c.D, t = threadIdx.x, lane = t & 63, wave = t >> 6;
    __shared__ float sm[2][kAttnWaves];
    __shared__ float so[kAttnWaves][256];
    const int64_t first = (int64_t)it.base * pl.hy + hk * pl.tiles + tile;
    auto ml = [&](int c, int which) { return pl.part_ml[(first + (int64_t)c * pl.hy) * 32 + which * 16 + n]; };
    float m = -INFINITY;
    for (int c = t; c < it.nc; c += kAttnThreads) m = fmaxf(m, ml(c, 0));
    for (int o = 32; o; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
    if (lane == 0) sm[0][wave] = m;
    __syncthreads();
    m = fmaxf(fmaxf(sm[0][0], sm[0][1]), fmaxf(sm[0][2], sm[0][3]));
    const float base = m == -INFINITY ? 0.0f : m;
    float l = 0.0f;
    for (int c = t; c < it.nc; c += kAttnThreads) l += ml(c, 1) * pow2(ml(c, 0) - base);
    for (int o = 32; o; o >>= 1) l += __shfl_xor(l, o);
    if (lane == 0) sm[1][wave] = l;
    float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int c = wave; c < it.nc; c += kAttnWaves) {
        const float f = pow2(ml(c, 0) - base);
        const float* o = pl.part_o + ((first + (int64_t)c * pl.hy) * 16 + n) * D;
#pragma unroll
        for (int x = 0; x < 4; ++x)
            if (lane + 64 * x < D) v[x] += f * o[lane + 64 * x];
    }
#pragma unroll
    for (int x = 0; x < 4; ++x) so[wave][lane + 64 * x] = v[x];
    __syncthreads();
    l = (sm[1][0] + sm[1][1]) + (sm[1][2] + sm[1][3]);
    if (t < D) {
        const float s = (so[0][t] + so[1][t]) + (so[2][t] + so[3][t]);
        a.out[it.row * a.ldo + (int64_t)h * D + t] = l == 0.0f ? 0.0f : s / l;
    }
    if (t == 0 && a.lse)
        a.lse[(int64_t)it.row * a.hq + h] = l == 0.0f ? -INFINITY : (m + log2f(l)) * 0.69314718056f;
}

// Adds the attention weights of a chunk to the scores: one workgroup per
// (item, kv head), every query head of the group.
__global__ __launch_bounds__(kAttnThreads) void attention_score_kernel(AttnArgs a, AttnPlan pl) {
    AttnItem it;
    if (!attn_plan(a, pl, blockIdx.x, false, &it)) return;
    const KvView& c = a.c;
    const int G = a.hq / c.hkv, hk = blockIdx.y, sq = a.seq ? a.seq[it.row] : it.row;
    extern __shared__ float hm[];  // [G] maximum, [G] 1 / sum
    for (int h = threadIdx.x; h < G; h += kAttnThreads) {
        const int64_t first = (int64_t)it.base * pl.hy + hk * pl.tiles + h / 16;
        float m = -INFINITY, l = 0.0f;
        for (int x = 0; x < it.nc; ++x) {
            const float* ml = pl.part_ml + (first + (int64_t)x * pl.hy) * 32 + h % 16;
            const float mn = fmaxf(m, ml[0]), base = mn == -INFINITY ? 0.0f : mn;
            l = l * pow2(m - base) + ml[16] * pow2(ml[0] - base);
            m = mn;
        }
        hm[h] = m == -INFINITY ? 0.0f : m;
        hm[G + h] = l == 0.0f ? 0.0f : 1.0f / l;
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

namespace {

AttnPlan make_plan(const AttnArgs& a, int cus, int64_t* items) {
    AttnPlan pl;
    const int G = a.hq / a.c.hkv;
    pl.part_o = pl.part_ml = pl.s = nullptr;
    pl.tiles = (G + 15) / 16;
    pl.hy = a.c.hkv * pl.tiles;
    const int64_t cap = (int64_t)a.c.max_pages * a.c.page;
    pl.cap = (cap + 31) / 32 * 32;
    // eight workgroups per compute unit, two at a time: the second half of
    // them evens out what differs between them
    const int64_t want = std::max<int64_t>(1, 8 * (int64_t)cus / pl.hy);
    pl.target = (int)want;
    pl.fixed = 0;
    if (a.R > kAttnPlanRows) {
        pl.fixed = (int)std::max<int64_t>(1, std::min<int64_t>(want / a.R, (cap + kAttnStep - 1) / kAttnStep));
        *items = a.R * pl.fixed;
    } else {
        // each row ends in a part of a chunk; no more chunks than positions
        *items = std::min(want + a.R, a.R * std::max<int64_t>(1, (cap + kAttnStep - 1) / kAttnStep));
    }
    return pl;
}

template <int DT>
hipError_t launch_attention(const AttnArgs& a, const AttnPlan& pl, int64_t items, hipStream_t s) {
    const dim3 grid((unsigned)items, (unsigned)pl.hy), block(kAttnThreads);
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
size_t place(const AttnArgs& a, int64_t items, AttnPlan* pl, char* base) {
    size_t at = 0;
    auto take = [&](size_t floats) {
        float* p = reinterpret_cast<float*>(base + at);
        at += (floats * 4 + 255) / 256 * 256;
        return p;
    };
    pl->part_ml = take((size_t)items * pl->hy * 32);
    pl->part_o = take((size_t)items * pl->hy * 16 * a.c.D);
    if (a.accumulate) pl->s = take((size_t)a.R * a.hq * pl->cap);
    return at;
}

}  // namespace

bool attention_joins(const AttnArgs& a, int cus) {
    int64_t items;
    const AttnPlan pl = make_plan(a, cus, &items);
    return items > a.R || a.accumulate || pl.fixed > 1;
}

size_t attention_workspace(const AttnArgs& a, int cus) {
    int64_t items;
    AttnPlan pl = make_plan(a, cus, &items);
    return place(a, items, &pl, nullptr);
}

hipError_t launch_paged_attention(int dtype, const AttnArgs& a, int cus, void* ws, hipStream_t s) {
    int64_t items;
    AttnPlan pl = make_plan(a, cus, &items);
    if (ws) (void)place(a, items, &pl, static_cast<char*>(ws));
    hipError_t e;
    switch (dtype) {
        case XT_F32: e = launch_attention<XT_F32>(a, pl, items, s); break;
        case XT_F16: e = launch_attention<XT_F16>(a, pl, items, s); break;
        default: e = launch_attention<XT_BF16>(a, pl, items, s); break;
    }
    if (e != hipSuccess) return e;
    if (items > a.R) {
        attention_join_kernel<<<dim3((unsigned)a.R, (unsigned)a.hq), kAttnThreads, 0, s>>>(a, pl);
        if ((e = hipGetLastError()) != hipSuccess) return e;
    }
    if (a.accumulate) {
        const size_t lds = 2 * sizeof(float) * (size_t)(a.hq / a.c.hkv);
        attention_score_kernel<<<dim3((unsigned)items, (unsigned)a.c.hkv), kAttnThreads, lds, s>>>(a, pl);
        e = hipGetLastError();
    }
    return e;
}

}  // namespace xt
