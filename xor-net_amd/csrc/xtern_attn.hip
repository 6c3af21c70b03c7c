// The paged key-value cache's append (rotary embedding, rounding, scatter)
// and the attention of one token per row over it.
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
// One workgroup per (row, query head), 256 positions at a time: a thread
// computes one position's s_j, then one column's share of the output.
constexpr int kAttnThreads = 256;

__device__ __forceinline__ float block_max(float v, float* sm) {
    for (int o = 32; o; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sm[threadIdx.x >> 6] = v;
    __syncthreads();
    return fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3]));
}
__device__ __forceinline__ float block_sum(float v, float* sm) {
    for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sm[threadIdx.x >> 6] = v;
    __syncthreads();
    return (sm[0] + sm[1]) + (sm[2] + sm[3]);
}

template <int DT>
__global__ __launch_bounds__(kAttnThreads) void paged_attention_kernel(AttnArgs a) {
    typedef Elem<DT> E;
    const KvView& c = a.c;
    const int64_t r = blockIdx.x;
    const int h = blockIdx.y, hk = h / (a.hq / c.hkv), t = threadIdx.x;
    __shared__ float sp[kAttnThreads];
    __shared__ int64_t so[kAttnThreads];
    __shared__ float sm[4];
    const int sq = a.seq ? a.seq[r] : (int)r;
    const int n = (unsigned)sq < (unsigned)c.nseq ? kv_length(c, a.lengths[r]) : 0;
    const float* q = a.q + r * a.ldq + (int64_t)h * c.D;
    const typename E::T* kc = static_cast<const typename E::T*>(c.k);
    const typename E::T* vc = static_cast<const typename E::T*>(c.v);
    float m = -INFINITY, l = 0.0f, o = 0.0f;
    auto score = [&](int p, int64_t* off, int* page) {
        *page = p < n ? kv_page(c, sq, p) : -1;
        *off = -1;
        if (*page < 0) return -INFINITY;
        *off = kv_offset(c, *page, p, hk);
        float acc = 0.0f;
        for (int d = 0; d < c.D; ++d) acc += q[d] * E::get(kc[*off + d]);
        return acc * a.scale;
    };
    for (int p0 = 0; p0 < n; p0 += kAttnThreads) {
        int64_t off;
        int pg;
        const float s = score(p0 + t, &off, &pg);
        const float mn = fmaxf(m, block_max(s, sm));
        const float base = mn == -INFINITY ? 0.0f : mn;
        const float f = expf(m - base);
        sp[t] = off < 0 ? 0.0f : expf(s - base);
        so[t] = off;
        m = mn;
        l = l * f + block_sum(sp[t], sm);
        o *= f;
        if (t < c.D) {
            const int cnt = min(kAttnThreads, n - p0);
            for (int j = 0; j < cnt; ++j)
                if (so[j] >= 0) o += sp[j] * E::get(vc[so[j] + t]);
        }
        __syncthreads();
    }
    if (t < c.D) a.out[r * a.ldo + (int64_t)h * c.D + t] = l == 0.0f ? 0.0f : o / l;
    const float lse = l == 0.0f ? -INFINITY : m + logf(l);
    if (a.lse && t == 0) a.lse[r * a.hq + h] = lse;
    if (!a.accumulate || l == 0.0f) return;
    for (int p = t; p < n; p += kAttnThreads) {
        int64_t off;
        int pg;
        const float s = score(p, &off, &pg);
        if (off >= 0) atomicAdd(&c.score[((int64_t)pg * c.hkv + hk) * c.page + p % c.page], expf(s - lse));
    }
}

hipError_t launch_paged_attention(int dtype, const AttnArgs& a, hipStream_t s) {
    const dim3 grid((unsigned)a.R, (unsigned)a.hq), block(kAttnThreads);
    switch (dtype) {
        case XT_F32: paged_attention_kernel<XT_F32><<<grid, block, 0, s>>>(a); break;
        case XT_F16: paged_attention_kernel<XT_F16><<<grid, block, 0, s>>>(a); break;
        default: paged_attention_kernel<XT_BF16><<<grid, block, 0, s>>>(a); break;
    }
    return hipGetLastError();
}

}  // namespace xt
