// New tokens into a paged cache with norms of their heads and, for a cache of
// 8-bit codes, a scale for each token and head; and cached positions read back.
#include <algorithm>

#include "xtern_cache.h"

namespace xt {

// A head x of D elements, of q and k with weights w and eps:
//   y_i = w_i x_i / sqrt(sum x^2 / D + eps)        (no norm: y = x)
// then the rotation of the pairs i, i + h as in kv_append_kernel; of v: y = x.
// q_out = y.  A cache of 8-bit codes holds y as c = round(y / s), s = a / 127
// rounded to f32, a = max |y| of the head as f32: |c| <= 127 and |c s - y| <=
// s / 2.  Below a = 2^-119 (1 / s would leave f32's normal numbers) s and c are
// 0; a head with an infinity or NaN has s = NaN, c = 0, so that what reads it
// sees NaN.
//
// All of it in 64 bits, then rounded to f32 and from there to a 16-bit cache's type;
// codes come from the 64 bits: a value
// next to the border of two codes falls where the exact one does, in whatever
// order sums are taken.  The f64 units take 4 cycles an instruction like the
// f32 ones, and a call is bound by its bytes or by its launch.
//
// A head is 16, 32 or 64 lanes of one wave, W = 4 elements each (D a multiple of
// four; no alignment is needed), or 64 lanes of every 64th element.  A lane also
// loads what its own elements are rotated with, OW = 4, 2 or 1 at a time as h is a
// multiple of these, and the next head's of both while it works on one.  The heads
// of a row go to several workgroups where rows are few.  HBM bounds long calls: 4096
// rows of 32 + 2 x 8 heads of 128 36 us (5.0 TB/s) on the same tensors again, 40.7 on
// others; one row takes 3.6.  Heads of 100:
// 34 us without a rotation, 36.5 with half of 25, 42.5 with 50 (element by element
// all of it: 54 and 66).
template <int DT> struct Held;
template <> struct Held<XT_I8> { typedef int8_t T; };
template <> struct Held<XT_F32> { typedef float T; };
template <> struct Held<XT_F16> { typedef _Float16 T; };
template <> struct Held<XT_BF16> { typedef __bf16 T; };

constexpr int kStoreThreads = 256;
constexpr float kLeastHead = 0x1p-119f;

// As lanes_sum.
template <int LANES>
__device__ __forceinline__ unsigned lanes_max(unsigned v) {
    v = max(v, (unsigned)dpp_to<0xb1>((int)v));
    v = max(v, (unsigned)dpp_to<0x4e>((int)v));
    v = max(v, (unsigned)dpp_to<0x141>((int)v));
    v = max(v, (unsigned)dpp_to<0x140>((int)v));
    if constexpr (LANES > 16) {
        const auto a = __builtin_amdgcn_permlane16_swap(v, v, false, false);
        v = max(a[0], a[1]);
    }
    if constexpr (LANES > 32) {
        const auto a = __builtin_amdgcn_permlane32_swap(v, v, false, false);
        v = max(a[0], a[1]);
    }
    return v;
}

template <int V> struct Width {
    static constexpr int value = V;
};

template <int DT, int W, int OW, int LANES>
__global__ __launch_bounds__(kStoreThreads) void kv_store_kernel(AppendArgs a) {
    typedef typename Held<DT>::T T;
    typedef float F4 __attribute__((ext_vector_type(4), aligned(4)));
    typedef float F2 __attribute__((ext_vector_type(2), aligned(4)));
    constexpr int kGroups = kStoreThreads / LANES;
    const KvView& c = a.c;
    const int64_t r = blockIdx.x;
    const int D = c.D, half = a.cos ? a.rot / 2 : 0, hq = a.q ? a.hq : 0, heads = hq + 2 * c.hkv;
    const int l = threadIdx.x & (LANES - 1), group = threadIdx.x / LANES;
    // element e of the lane; what it is rotated with, and by which pair
    int d[4], other[4], pair[4];
    bool turns[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        d[e] = W == 4 ? 4 * l + e : l + 64 * e;
        turns[e] = d[e / OW * OW] < 2 * half;  // (OW of them turn together)
        other[e] = !turns[e] ? d[e] : (d[e] < half ? d[e] + half : d[e] - half);
        pair[e] = !turns[e] ? 0 : (d[e] < half ? d[e] : d[e] - half);
    }
    const bool any = W == 4 ? d[0] < D : true;  // (W 4: all four or none)
    // The four elements at i[0], or two each at i[0] and i[2], side by side, or those
    // of the four that are of the head
    auto get = [&](auto width, const float* p, const int* i, float* x) {
        constexpr int V = decltype(width)::value;
        if constexpr (V == 2) {
#pragma unroll
            for (int e = 0; e < 4; e += 2) {
                const F2 v = *reinterpret_cast<const F2*>(p + (any ? i[e] : 0));
                x[e] = v[0];
                x[e + 1] = v[1];
            }
        } else if constexpr (V == 4) {
            const F4 v = *reinterpret_cast<const F4*>(p + (any ? i[0] : 0));
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = v[e];
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = d[e] < D ? p[i[e]] : 0.0f;
        }
    };
    // x of head h, and what it is rotated with
    auto load = [&](int h, float* x, float* z) {
        const bool isq = h < hq, isv = h >= hq + c.hkv;
        const float* src = (isq ? a.q + r * a.ldq + (int64_t)h * D
                                : (isv ? a.v + r * a.ldv + (int64_t)(h - hq - c.hkv) * D
                                       : a.k + r * a.ldk + (int64_t)(h - hq) * D));
        get(Width<W>{}, src, d, x);
        if (half && !isv) get(Width<OW>{}, src, other, z);
    };
    const int step = gridDim.y * kGroups;
    int h = blockIdx.y * kGroups + group;
    float x[4], z[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (h < heads) load(h, x, z);  // (with the row's place still on its way)
    const int slot = a.slots[r];
    const int sq = a.seq ? a.seq[r] : (int)r;
    const int pos = a.cos ? a.pos[r] : 0;
    int pg = -1;
    if (slot >= 0 && slot < (int64_t)c.max_pages * c.page && (unsigned)sq < (unsigned)c.nseq &&
        (!a.cos || (pos >= 0 && pos < a.rope_rows)))
        pg = kv_page(c, sq, slot);
    if (a.lengths && blockIdx.y == 0 && threadIdx.x == 0) a.lengths[r] = pg < 0 ? 0 : slot + 1;
    if (pg < 0) return;
    if (c.score && blockIdx.y == 0)
        for (int i = threadIdx.x; i < c.hkv; i += kStoreThreads)
            c.score[((int64_t)pg * c.hkv + i) * c.page + kv_slot(c, slot)] = 0.0f;
    const int64_t at = kv_offset(c, pg, slot, 0);
    // Norm and rotation of an element as inv (x A + z B), z what it is rotated
    // with: A = w cos, B = w' (-sin or sin); of q and of k
    double A[2][4], B[2][4];
    {
        float cs[4], sn[4], w[2][4], o[2][4];
        if (half) {
            get(Width<OW>{}, a.cos + (int64_t)pos * half, pair, cs);
            get(Width<OW>{}, a.sin + (int64_t)pos * half, pair, sn);
        }
        if (a.k_norm) {
            get(Width<W>{}, a.k_norm, d, w[1]);
            get(Width<OW>{}, a.k_norm, other, o[1]);
            if (hq) {
                get(Width<W>{}, a.q_norm, d, w[0]);
                get(Width<OW>{}, a.q_norm, other, o[0]);
            }
        }
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                A[i][e] = a.k_norm ? (double)w[i][e] : 1.0;
                B[i][e] = 0.0;
                if (turns[e]) {
                    B[i][e] = (a.k_norm ? (double)o[i][e] : 1.0) * (d[e] < half ? -sn[e] : sn[e]);
                    A[i][e] *= cs[e];
                }
            }
    }
#pragma unroll 1
    for (; h < heads; h += step) {
        float nx[4], nz[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        if (h + step < heads) load(h + step, nx, nz);
        const bool isq = h < hq, isv = h >= hq + c.hkv;
        const int head = isq ? h : (isv ? h - hq - c.hkv : h - hq);
        double y[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = any ? x[e] : 0.0f;
        if (!isv) {
            double inv = 1.0;
            if (a.k_norm) {
                // (the root from the hardware's estimate, 2^-23, in two steps)
                const double v = lanes_sum<LANES>(fma(y[0], y[0], fma(y[1], y[1], fma(y[2], y[2], y[3] * y[3])))) * a.inv_dim +
                                 a.eps;
                inv = __builtin_amdgcn_rsq(v);
                inv = fma(inv * 0.5, fma(-v * inv, inv, 1.0), inv);
                inv = fma(inv * 0.5, fma(-v * inv, inv, 1.0), inv);
                if (!(v > 0.0 && v < INFINITY)) inv = 1.0 / sqrt(v);  // (0, infinity, NaN)
            }
#pragma unroll
            for (int e = 0; e < 4; ++e)
                y[e] = fma(y[e], isq ? A[0][e] : A[1][e], (turns[e] ? (double)z[e] : 0.0) * (isq ? B[0][e] : B[1][e])) * inv;
        }
        float f[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            f[e] = (float)y[e];
            x[e] = nx[e];
            z[e] = nz[e];
        }
        if (isq) {
            float* to = a.qo + r * a.ldqo + (int64_t)head * D;
            if constexpr (W == 4) {
                if (any) *reinterpret_cast<F4*>(to + d[0]) = F4{f[0], f[1], f[2], f[3]};
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (d[e] < D) to[d[e]] = f[e];
            }
            continue;
        }
        T* to = static_cast<T*>(isv ? c.v : c.k) + at + head * c.sh;
        T held[4];
        if constexpr (DT == XT_I8) {
            unsigned top = 0;  // (as whole numbers: NaN above infinity above the rest)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (d[e] < D) top = max(top, __float_as_uint(f[e]) & 0x7fffffffu);
            const float m = __uint_as_float(lanes_max<LANES>(top));
            const bool zero = !(m >= kLeastHead && m < INFINITY);  // (or NaN)
            // (m has 24 bits: m / 127 is 2^-32 or more from the middle of two floats,
            // so that the product rounds like the quotient)
            const float scale = m < kLeastHead ? 0.0f : (m < INFINITY ? (float)((double)m * (1.0 / 127.0)) : NAN);
            double up = __builtin_amdgcn_rcp((double)scale);  // (2^-23, in a step 2^-46)
            up = fma(up, fma(-(double)scale, up, 1.0), up);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                // The quotient, not the product with its divisor's reciprocal: that one
                // misses middles between two codes (73.5 / 49, whose code is 2, gives
                // 1.4999999999999998).  One correction, with what the product leaves of
                // y: 2^-92, so a quotient of 53 bits comes out as it is.
                double n = y[e] * up;
                n = fma(fma(-n, (double)scale, y[e]), up, n);
                held[e] = zero ? 0 : (int8_t)(int)rint(n);
            }
            if (l == 0) (isv ? a.vs : a.ks)[((int64_t)pg * c.hkv + head) * c.page + kv_slot(c, slot)] = scale;
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) held[e] = Elem<DT>::put(f[e]);
        }
        if constexpr (W == 4) {
            typedef T V __attribute__((ext_vector_type(4)));
            typedef V U __attribute__((aligned(sizeof(T))));
            if (any) *reinterpret_cast<U*>(to + d[0]) = V{held[0], held[1], held[2], held[3]};
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (d[e] < D) to[d[e]] = held[e];
        }
    }
}

// Rows r of k and v: position slots[r] of its sequence, codes times their scale
// (or elements) rounded to the output's type; zeros for a row that names no
// position.  Bound by HBM: a workgroup takes N rows, whose places N threads look
// up side by side, then copies them, W elements (16 bytes of output) a thread and
// four rows of it at once: 65536 positions of 8 heads of 128 to bf16 85 us (4.8 TB/s
// read and written; one row at once 93), 41493 of 5 of 192 to f32 88 (128).
template <int DT, int OT, int W>
__global__ __launch_bounds__(256) void kv_read_kernel(ReadArgs a, int rows) {
    typedef typename Held<DT>::T T;
    typedef typename Elem<OT>::T O;
    const KvView& c = a.c;
    constexpr int kMost = 32;
    __shared__ int64_t off[kMost], sc[kMost];
    const int64_t r0 = (int64_t)blockIdx.x * rows;
    const int n = (int)min((int64_t)rows, a.R - r0);
    if ((int)threadIdx.x < n) {
        const int64_t r = r0 + threadIdx.x;
        const int slot = a.slots[r], sq = a.seq ? a.seq[r] : (int)r;
        int pg = -1;
        if (slot >= 0 && slot < (int64_t)c.max_pages * c.page && (unsigned)sq < (unsigned)c.nseq) pg = kv_page(c, sq, slot);
        off[threadIdx.x] = pg < 0 ? -1 : kv_offset(c, pg, slot, 0);
        sc[threadIdx.x] = pg < 0 ? 0 : (int64_t)pg * c.hkv * c.page + kv_slot(c, slot);
    }
    __syncthreads();
    const int per = c.D / W, row = c.hkv * per, both = 2 * row;
    // threads of a row: as many as it has pieces, rounded up to a power of two
    const int lg = min(8, 32 - __builtin_clz(both - 1)), step = 256 >> lg;
    typedef T V __attribute__((ext_vector_type(W)));
    typedef V VU __attribute__((aligned(sizeof(T))));
    typedef O X __attribute__((ext_vector_type(W)));
    typedef X XU __attribute__((aligned(sizeof(O))));
    constexpr int U = 4;  // rows of a thread on their way
    for (int x0 = threadIdx.x >> lg; x0 < n; x0 += U * step) {
        int64_t from[U], sat[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int x = min(x0 + u * step, n - 1);
            from[u] = off[x];
            sat[u] = sc[x];
        }
        for (int j = threadIdx.x & ((1 << lg) - 1); j < both; j += 1 << lg) {
            const bool isv = j >= row;
            const int k = isv ? j - row : j, h = fast_quot(k, a.by_per), e = (k - h * per) * W;
            O* out = static_cast<O*>(isv ? a.v : a.k) + (int64_t)h * c.D + e;
            const T* in = static_cast<const T*>(isv ? c.v : c.k) + h * c.sh + e;
            [[maybe_unused]] const float* scales = (isv ? a.vs : a.ks) + (int64_t)h * c.page;
            const int64_t ld = isv ? a.ldv : a.ldk;
            V v[U];
            [[maybe_unused]] float s[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {  // (no position: the first one, and not used)
                v[u] = *reinterpret_cast<const VU*>(in + max(from[u], (int64_t)0));
                if constexpr (DT == XT_I8) s[u] = scales[sat[u]];
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (x0 + u * step >= n) break;
                X y;
#pragma unroll
                for (int i = 0; i < W; ++i) {
                    if constexpr (DT == XT_I8) {
                        float f = s[u] * (float)v[u][i];
                        // (an f32 of its own: with one element a thread the
                        // compiler would round the product to f16 at once)
                        asm("" : "+v"(f));
                        y[i] = Elem<OT>::put(from[u] < 0 ? 0.0f : f);
                    } else {
                        y[i] = Elem<OT>::put(from[u] < 0 ? 0.0f : Elem<DT>::get(v[u][i]));
                    }
                }
                *reinterpret_cast<XU*>(out + (r0 + x0 + u * step) * ld) = y;
            }
        }
    }
}

namespace {

template <int DT, int OW>
void launch_store_of(const AppendArgs& a, int lanes, dim3 grid, hipStream_t s) {
    if (lanes == 64)
        kv_store_kernel<DT, 4, OW, 64><<<grid, kStoreThreads, 0, s>>>(a);
    else if (lanes == 32)
        kv_store_kernel<DT, 4, OW, 32><<<grid, kStoreThreads, 0, s>>>(a);
    else
        kv_store_kernel<DT, 4, OW, 16><<<grid, kStoreThreads, 0, s>>>(a);
}

template <int DT>
hipError_t launch_store(AppendArgs& a, int cus, hipStream_t s) {
    const int half = a.cos ? a.rot / 2 : 0, D = a.c.D;
    const bool wide = D % 4 == 0;
    a.inv_dim = 1.0 / D;
    const int lanes = !wide || D > 128 ? 64 : (D > 64 ? 32 : 16), groups = kStoreThreads / lanes;
    const int64_t heads = (a.q ? a.hq : 0) + 2 * (int64_t)a.c.hkv;
    // workgroups of a row: until two per compute unit (77 rows of 32 + 64 heads: 5.8
    // us, until four 6.1, eight 6.2)
    const int64_t want = std::max<int64_t>(1, 2 * (int64_t)cus / a.R);
    const dim3 grid((unsigned)a.R, (unsigned)std::min((heads + groups - 1) / groups, want));
    if (!wide)
        kv_store_kernel<DT, 1, 1, 64><<<grid, kStoreThreads, 0, s>>>(a);
    else if (half % 4 == 0)
        launch_store_of<DT, 4>(a, lanes, grid, s);
    else if (half % 2 == 0)
        launch_store_of<DT, 2>(a, lanes, grid, s);
    else
        launch_store_of<DT, 1>(a, lanes, grid, s);
    return hipGetLastError();
}

template <int DT, int OT>
hipError_t launch_read(ReadArgs& a, int cus, hipStream_t s) {
    constexpr int kWide = OT == XT_F32 ? 4 : 8;
    const int w = a.c.D % kWide == 0 ? kWide : (a.c.D % 4 == 0 ? 4 : 1);
    a.by_per = fast_div(a.c.D / w);
    const int64_t both = 2 * (int64_t)a.c.hkv * (a.c.D / w);
    // rows until four workgroups per compute unit, or 16 pieces a thread (until
    // eight / 16: 4096 positions of 8 heads of 128 7.1 / 8.7 us, here 6.6)
    const int rows = (int)std::max<int64_t>(
        1, std::min<int64_t>(std::min<int64_t>(32, 4096 / both), a.R / (4 * (int64_t)cus)));
    const unsigned grid = (unsigned)((a.R + rows - 1) / rows);
    if (w == kWide)
        kv_read_kernel<DT, OT, kWide><<<grid, 256, 0, s>>>(a, rows);
    else if (w == 4)
        kv_read_kernel<DT, OT, 4><<<grid, 256, 0, s>>>(a, rows);
    else
        kv_read_kernel<DT, OT, 1><<<grid, 256, 0, s>>>(a, rows);
    return hipGetLastError();
}

template <int DT>
hipError_t launch_read_as(int out, ReadArgs& a, int cus, hipStream_t s) {
    switch (out) {
        case XT_F32: return launch_read<DT, XT_F32>(a, cus, s);
        case XT_F16: return launch_read<DT, XT_F16>(a, cus, s);
        default: return launch_read<DT, XT_BF16>(a, cus, s);
    }
}

}  // namespace

hipError_t launch_kv_store(int dtype, AppendArgs a, int cus, hipStream_t s) {
    switch (dtype) {
        case XT_F32: return launch_store<XT_F32>(a, cus, s);
        case XT_F16: return launch_store<XT_F16>(a, cus, s);
        case XT_BF16: return launch_store<XT_BF16>(a, cus, s);
        default: return launch_store<XT_I8>(a, cus, s);
    }
}

hipError_t launch_kv_read(int dtype, int out, ReadArgs a, int cus, hipStream_t s) {
    switch (dtype) {
        case XT_F32: return launch_read_as<XT_F32>(out, a, cus, s);
        case XT_F16: return launch_read_as<XT_F16>(out, a, cus, s);
        case XT_BF16: return launch_read_as<XT_BF16>(out, a, cus, s);
        default: return launch_read_as<XT_I8>(out, a, cus, s);
    }
}

}  // namespace xt
