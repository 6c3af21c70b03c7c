// Token probabilities of rows of logits: ln p of given tokens, entropy, the
// most likely tokens.
//
// m = max x, z = sum over all but one maximum of exp(x - m),
// ln p(t) = x_t - m - ln(1 + z), H = ln(1 + z) - sum (x - m) exp(x - m) / (1 + z).
// Leaving the maximum's own 1 out of the sum keeps ln p of an almost certain
// token exact to its last bits.  Logits of -inf have p = 0; a row of nothing
// else gives ln p = -inf and H = 0.
#include "xtern_cache.h"
#include "xtern_device.h"

namespace xt {

constexpr int kProbsThreads = 1024;

// Order of the alternatives: larger value first, then the lower index; NaN
// behind everything.
__device__ __forceinline__ unsigned long long probs_key(float x, int i) {
    const float f = x + 0.0f;  // (-0 counts as +0)
    unsigned u = __float_as_uint(f);
    u = f != f ? 0u : u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u);
    return ((unsigned long long)u << 32) | (unsigned)~i;
}

template <typename T, typename Op>
__device__ __forceinline__ T wg_reduce(T v, T* sm, Op op) {
    for (int o = 32; o; o >>= 1) v = op(v, (T)__shfl_xor(v, o));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sm[threadIdx.x >> 6] = v;
    __syncthreads();
    v = sm[0];
    for (int w = 1; w < kProbsThreads / 64; ++w) v = op(v, sm[w]);
    return v;
}

template <int DT>
__global__ __launch_bounds__(kProbsThreads) void token_logprobs_kernel(ProbsArgs a) {
    typedef Elem<DT> E;
    const int64_t r = blockIdx.x;
    const int t = threadIdx.x;
    const typename E::T* x = static_cast<const typename E::T*>(a.x) + r * a.ld;
    __shared__ float smf[16];
    __shared__ unsigned long long smk[16];
    auto add = [](float p, float q) { return p + q; };
    auto top = [](unsigned long long p, unsigned long long q) { return p > q ? p : q; };
    unsigned long long best = 0;
    for (int i = t; i < a.V; i += kProbsThreads) {
        const unsigned long long k = probs_key(E::get(x[i]), i);
        best = top(best, k);
    }
    best = wg_reduce(best, smk, top);
    const int imax = (int)~(unsigned)best;
    const float m = E::get(x[imax]);
    float z = 0.0f, xz = 0.0f;
    for (int i = t; i < a.V; i += kProbsThreads) {
        const float v = E::get(x[i]), d = v - m;
        if (i == imax || v == -INFINITY) continue;
        const float e = expf(d);
        z += e;
        xz += d * e;
    }
    z = wg_reduce(z, smf, add);
    xz = wg_reduce(xz, smf, add);
    const bool none = m == -INFINITY && z == z;  // (a NaN beside them makes the row NaN)
    const float bad = m == INFINITY ? NAN : 0.0f;
    const float ln = log1pf(z) + bad;
    if (t == 0) a.entropy[r] = none ? 0.0f : ln - xz / (1.0f + z);
    for (int i = t; i < a.T; i += kProbsThreads) {
        const int tok = a.tokens[r * a.T + i];
        float lp = tok < 0 ? 0.0f : NAN;
        if (tok >= 0 && tok < a.V) lp = none ? E::get(x[tok]) : E::get(x[tok]) - m - ln;
        a.lp[r * a.T + i] = lp;
    }
    for (int j = 0; j < a.top; ++j) {
        if (t == 0) {
            const int i = (int)~(unsigned)best;
            a.ids[r * a.top + j] = i;
            a.top_lp[r * a.top + j] = none ? E::get(x[i]) : E::get(x[i]) - m - ln;
        }
        unsigned long long next = 0;
        for (int i = t; i < a.V; i += kProbsThreads) {
            const unsigned long long k = probs_key(E::get(x[i]), i);
            if (k < best) next = top(next, k);
        }
        best = wg_reduce(next, smk, top);
    }
}

hipError_t launch_token_logprobs(int dtype, const ProbsArgs& a, hipStream_t s) {
    const dim3 grid((unsigned)a.M), block(kProbsThreads);
    switch (dtype) {
        case XT_F32: token_logprobs_kernel<XT_F32><<<grid, block, 0, s>>>(a); break;
        case XT_F16: token_logprobs_kernel<XT_F16><<<grid, block, 0, s>>>(a); break;
        default: token_logprobs_kernel<XT_BF16><<<grid, block, 0, s>>>(a); break;
    }
    return hipGetLastError();
}

}  // namespace xt
