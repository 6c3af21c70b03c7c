// Verification of drafted tokens: which of them the target's probabilities
// accept, and the token that follows the last one that was.
//
// With p_t the target's and q_t the draft's probabilities at place t (softmax of
// the logits over the temperature; without draft logits all of q_t lies on the
// drafted token), drafted tokens x_t and given u_t in [0, 1): x_0 .. x_{n-1} are
// accepted, n the first t with u_t q_t(x_t) >= p_t(x_t), or the number of drafts.
// The token after them is drawn from max(p_n - q_n, 0), or from p_n where all
// drafts were accepted (or nothing is left of it): the first i whose sum up to i
// is above u_T times the whole.  So the tokens are distributed as the target's.
// At temperature 0 everything lies on the largest logit, the lowest of equals.
//
// Everything that decides is in 64 bits: a token flips where a sum of V terms
// crosses a border, and f32 exponentials would move some of V borders by 1e-8
// each.  The first kernel reads every row that can count once (HBM bounds large
// calls: f64 instructions go at the rate of f32 ones), rows cut into slices
// where they are few; the second decides, reads the one row that is drawn from
// again, in tiles of 1024 logits a wave, and the workgroup that ends the
// sequence's last tile finds the tile and in it the token (sums and count at
// device scope, as the chip's eight L2s need it).
#include <algorithm>

#include "xtern_cache.h"

namespace xt {

constexpr int kVerifyThreads = 256;
constexpr int kVerifyWaves = kVerifyThreads / 64;
constexpr int kVerifyPer = 16;                     // logits of a lane and tile
constexpr int kVerifyTile = 64 * kVerifyPer;       // of a wave
constexpr int kVerifyRows = 2 * kVerifyDrafts + 1; // of a sequence: target, then draft
constexpr int kVerifySlices = 64;

// A slice of a row: l = sum exp((x - m) / temperature), m its maximum; `at`
// (temperature 0): the first index of m.  What is no probability (NaN, +inf)
// gives l = NaN.
struct RowStat {
    double l;
    float m;
    int at;
};

struct VerifyPlan {
    RowStat* stats;   // [S][rows][slices]
    double* sums;     // [S][tiles]
    unsigned* count;  // [S]: workgroups done, zero between calls
    int rows;         // of a sequence: T + 1, and T of the draft
    int slices, tiles, blocks;
};

__device__ __forceinline__ float verify_temp(const VerifyArgs& a, int b) {
    return a.temps ? a.temps[b] : a.temp;
}
// Drafts of sequence b; negative: the sequence is not there.
__device__ __forceinline__ int verify_count(const VerifyArgs& a, int b) {
    return a.counts ? min(a.counts[b], a.T) : a.T;
}
template <typename T>
__device__ __forceinline__ const T* verify_row(const VerifyArgs& a, int b, int j) {
    return j <= a.T ? static_cast<const T*>(a.target) + b * a.ld_seq + j * a.ld_row
                    : static_cast<const T*>(a.draft) + b * a.ldd_seq + (j - a.T - 1) * a.ldd_row;
}

// exp((x - m) / temperature) for x <= m, c = log2 e / temperature: with y = (x -
// m) c = n + f, |f| <= 1/2, 2^n times a polynomial of 2^f, of degree 9 through its
// values in Chebyshev's nodes (the constant term then made 1, so that m itself
// gives 1): 3e-14 of the result.  0 for x = -inf; the caller sees to NaN and +inf.
__device__ __forceinline__ double verify_exp(float x, float m, double c) {
    const double y = fmax(((double)x - (double)m) * c, -1100.0);
    const double magic = 0x1.8p52, z = y + magic;  // (its last bits: n)
    const double f = y - (z - magic);
    double p = 0x1.b6571de2f2351p-24;
    p = fma(p, f, 0x1.63ef969a64d3cp-20);
    p = fma(p, f, 0x1.ffcb76789860fp-17);
    p = fma(p, f, 0x1.43088e257f341p-13);
    p = fma(p, f, 0x1.5d87fe908f88ap-10);
    p = fma(p, f, 0x1.3b2ab72b175eep-7);
    p = fma(p, f, 0x1.c6b08d7044119p-5);
    p = fma(p, f, 0x1.ebfbdff8149f2p-3);
    p = fma(p, f, 0x1.62e42fefa39f7p-1);
    p = fma(p, f, 1.0);
    return ldexp(p, (int)__builtin_bit_cast(int64_t, z));
}
__device__ __forceinline__ double verify_rate(float temp) {
    return temp > 0.0f ? 1.4426950408889634 / (double)temp : 0.0;
}

// A lane's logits of a tile: vectors of 16 bytes (W logits), vector v at base +
// (v * 64 + lane) * W; -inf past the row.
template <int DT>
struct VerifyTile {
    static constexpr int W = DT == XT_F32 ? 4 : 8, NV = kVerifyPer / W;
    typedef typename Elem<DT>::T T;
    typedef T Vec __attribute__((ext_vector_type(W)));
    typedef Vec VecU __attribute__((aligned(sizeof(T))));
    float x[kVerifyPer];
    __device__ __forceinline__ static int index(int base, int i) {
        return base + ((i / W) * 64 + (int)(threadIdx.x & 63)) * W + i % W;
    }
    __device__ __forceinline__ void load(const T* row, int base, int V) {
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int at = index(base, v * W);
            Vec q;
            if (at + W <= V) {
                q = *reinterpret_cast<const VecU*>(row + at);
            } else {
#pragma unroll
                for (int j = 0; j < W; ++j) q[j] = at + j < V ? row[at + j] : (T)-INFINITY;
            }
#pragma unroll
            for (int j = 0; j < W; ++j) x[v * W + j] = Elem<DT>::get(q[j]);
        }
    }
};

__device__ __forceinline__ double wave_add(double v) {
    for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
    return v;
}
__device__ __forceinline__ float wave_most(float v) {
    for (int o = 32; o; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));
    return v;
}
__device__ __forceinline__ int wave_least(int v) {
    for (int o = 32; o; o >>= 1) v = min(v, __shfl_xor(v, o));
    return v;
}

// Joins stats of one a lane (neutral: l 0, m -inf).
__device__ __forceinline__ RowStat wave_join(RowStat s, double c) {
    const float m = wave_most(s.m);
    RowStat r;
    r.at = wave_least(s.m == m ? s.at : 0x7fffffff);
    r.l = wave_add(s.m == -INFINITY && s.l == 0.0 ? 0.0 : (m == -INFINITY ? s.l : s.l * verify_exp(s.m, m, c)));
    r.m = m;
    return r;
}

template <int DT>
__global__ __launch_bounds__(kVerifyThreads) void verify_stats_kernel(VerifyArgs a, VerifyPlan pl) {
    typedef VerifyTile<DT> R;
    __shared__ RowStat waves[kVerifyWaves];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int slice = blockIdx.x % pl.slices, row = blockIdx.x / pl.slices, b = row / pl.rows, j = row % pl.rows;
    const int count = verify_count(a, b);
    if (j <= a.T ? j > count : j - a.T - 1 >= count) return;
    const float temp = verify_temp(a, b);
    const double c = verify_rate(temp);
    const typename R::T* x = verify_row<typename R::T>(a, b, j);
    const int per = (pl.tiles + pl.slices - 1) / pl.slices, t1 = min(pl.tiles, (slice + 1) * per);
    RowStat s{0.0, -INFINITY, 0x7fffffff};
    bool bad = false;
    for (int t = slice * per + wave; t < t1; t += kVerifyWaves) {
        R r;
        r.load(x, t * kVerifyTile, a.V);
        float m = s.m;
#pragma unroll
        for (int i = 0; i < kVerifyPer; ++i) {
            m = fmaxf(m, r.x[i]);
            bad |= !(r.x[i] < INFINITY);
        }
        if (temp > 0.0f) {
            if (m > s.m) {
                s.l *= s.m == -INFINITY ? 0.0 : verify_exp(s.m, m, c);
                s.m = m;
            }
            const float base = s.m == -INFINITY ? 0.0f : s.m;
#pragma unroll
            for (int i = 0; i < kVerifyPer; ++i) s.l += verify_exp(r.x[i], base, c);
        } else {
            if (m > s.m) {
                int at = 0x7fffffff;
#pragma unroll
                for (int i = kVerifyPer - 1; i >= 0; --i)
                    if (r.x[i] == m) at = R::index(t * kVerifyTile, i);
                s.m = m;
                s.at = at;
            }
        }
    }
    if (bad) s.l = NAN;
    s = wave_join(s, c);
    if (lane == 0) waves[wave] = s;
    __syncthreads();
    if (wave == 0) {
        s = lane < kVerifyWaves ? waves[lane] : RowStat{0.0, -INFINITY, 0x7fffffff};
        s = wave_join(s, c);
        if (lane == 0) pl.stats[(int64_t)row * pl.slices + slice] = s;
    }
}

// What the second kernel draws from: max(p - q, 0), each exp((x - m) / temperature) / l.
struct VerifyDraw {
    float pm, qm;
    double pl, ql;  // 1 / l
    double c;
    int one;        // all of q: this token (draft NULL), -1: none of it
    bool draft;     // q of the draft's logits
};
template <int DT>
__device__ __forceinline__ void verify_left(const VerifyDraw& w, const VerifyTile<DT>& p, const VerifyTile<DT>& q,
                                            int base, double* left) {
#pragma unroll
    for (int i = 0; i < kVerifyPer; ++i) {
        double v = verify_exp(p.x[i], w.pm, w.c) * w.pl;
        if (w.draft) v = fmax(v - verify_exp(q.x[i], w.qm, w.c) * w.ql, 0.0);
        if (VerifyTile<DT>::index(base, i) == w.one) v = 0.0;
        left[i] = v;
    }
}

__device__ __forceinline__ void st_device(double* p, double v) {
    __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ double ld_device(const double* p) {
    return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// Sums of the tiles first, first + step, ... of what is left.
template <int DT>
__device__ void verify_sums(const VerifyArgs& a, const VerifyPlan& pl, const VerifyDraw& w, int b, int n, int first,
                            int step) {
    typedef VerifyTile<DT> R;
    const typename R::T* prow = verify_row<typename R::T>(a, b, n);
    const typename R::T* qrow = w.draft ? verify_row<typename R::T>(a, b, a.T + 1 + n) : prow;
    for (int t = first; t < pl.tiles; t += step) {
        R p, q;
        p.load(prow, t * kVerifyTile, a.V);
        if (w.draft) q.load(qrow, t * kVerifyTile, a.V);
        double left[kVerifyPer], sum = 0.0;
        verify_left<DT>(w, p, q, t * kVerifyTile, left);
#pragma unroll
        for (int i = 0; i < kVerifyPer; ++i) sum += left[i];
        sum = wave_add(sum);
        if ((threadIdx.x & 63) == 0) st_device(pl.sums + (int64_t)b * pl.tiles + t, sum);
    }
}

template <int DT>
__global__ __launch_bounds__(kVerifyThreads) void verify_draw_kernel(VerifyArgs a, VerifyPlan pl) {
    typedef VerifyTile<DT> R;
    typedef typename R::T T;
    __shared__ RowStat rows[kVerifyRows];
    __shared__ double chunk[kVerifyThreads];
    __shared__ double ends[kVerifyWaves];
    __shared__ int lds_n, lds_last, lds_tile, lds_first;
    __shared__ double lds_total, lds_before;
    const int b = blockIdx.x / pl.blocks, block = blockIdx.x % pl.blocks;
    const int t = threadIdx.x, wave = t >> 6, lane = t & 63;
    const int count = verify_count(a, b);
    const float temp = verify_temp(a, b);
    const double c = verify_rate(temp);
    const bool there = count >= 0 && temp >= 0.0f && temp < INFINITY;
    // the rows' sums
    for (int j = wave; there && j < pl.rows; j += kVerifyWaves) {
        if (j <= a.T ? j > count : j - a.T - 1 >= count) continue;
        RowStat s{0.0, -INFINITY, 0x7fffffff};
        if (lane < pl.slices) s = pl.stats[((int64_t)b * pl.rows + j) * pl.slices + lane];
        s = wave_join(s, c);
        if (temp == 0.0f) s.l = s.m == -INFINITY ? NAN : s.l + 1.0;
        if (lane == 0) rows[j] = s;
    }
    __syncthreads();
    // a row of probabilities: its sum is a number, and not 0
    auto fine = [&](int j) { return rows[j].l > 0.0 && rows[j].l < INFINITY; };
    auto chance = [&](int j, float x) { return verify_exp(x, rows[j].m, c) / rows[j].l; };
    if (wave == 0) {
        // lane t: whether draft t is accepted
        bool taken = false;
        if (there && lane < count) {
            const int x = a.drafted[(int64_t)b * a.T + lane];
            const float u = a.uniforms[(int64_t)b * (a.T + 1) + lane];
            if (x >= 0 && x < a.V && fine(lane) && (!a.draft || fine(a.T + 1 + lane))) {
                if (temp == 0.0f) {
                    taken = x == rows[lane].at;
                } else {
                    const double p = chance(lane, Elem<DT>::get(verify_row<T>(a, b, lane)[x]));
                    const double q = a.draft ? chance(a.T + 1 + lane, Elem<DT>::get(verify_row<T>(a, b, a.T + 1 + lane)[x])) : 1.0;
                    taken = (double)u * q < p;
                }
            }
        }
        const uint64_t no = ~__ballot(taken);
        if (lane == 0) lds_n = there ? min(no ? (int)__builtin_ctzll(no) : 64, count) : 0;
    }
    __syncthreads();
    const int n = lds_n;
    // the draft that was not accepted; none, or one that is no token: all of p is left
    const int x = there && n < count ? a.drafted[(int64_t)b * a.T + n] : -1;
    const bool refused = x >= 0 && x < a.V;
    const bool drawn = there && fine(n) && !(refused && a.draft && !fine(a.T + 1 + n));
    auto finish = [&](int token) {
        if (t == 0) a.accepted[b] = n;
        for (int i = t; i <= a.T; i += kVerifyThreads) {
            const int64_t at = (int64_t)b * (a.T + 1) + i;
            const int id = i < n ? a.drafted[(int64_t)b * a.T + i] : (i == n ? token : -1);
            a.tokens[at] = id;
            float lp = 0.0f;
            if (id >= 0 && temp > 0.0f)
                lp = (float)(((double)Elem<DT>::get(verify_row<T>(a, b, i)[id]) - (double)rows[i].m) / (double)temp - log(rows[i].l));
            a.logprobs[at] = lp;
        }
    };
    if (!drawn || temp == 0.0f) {
        if (block == 0) finish(drawn ? rows[n].at : -1);
        return;
    }
    VerifyDraw w;
    w.pm = rows[n].m;
    w.pl = 1.0 / rows[n].l;
    w.c = c;
    w.draft = refused && a.draft;
    w.one = refused && !a.draft ? x : -1;
    w.qm = w.draft ? rows[a.T + 1 + n].m : 0.0f;
    w.ql = w.draft ? 1.0 / rows[a.T + 1 + n].l : 0.0;
    verify_sums<DT>(a, pl, w, b, n, block * kVerifyWaves + wave, pl.blocks * kVerifyWaves);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // every store has arrived
    __syncthreads();
    // (the count wraps to zero by itself, for the next call)
    if (t == 0) lds_last = atomicInc(pl.count + b, (unsigned)pl.blocks - 1) == (unsigned)pl.blocks - 1;
    __syncthreads();
    if (!lds_last) return;
    // The tile: a run of tiles a thread, the sums before each thread
    const int per = (pl.tiles + kVerifyThreads - 1) / kVerifyThreads, first = t * per, end = min(pl.tiles, first + per);
    const double* sums = pl.sums + (int64_t)b * pl.tiles;
    const double u = a.uniforms[(int64_t)b * (a.T + 1) + a.T];
    for (int pass = 0; pass < 2; ++pass) {
        double mine = 0.0;
        for (int i = first; i < end; ++i) mine += ld_device(sums + i);
        double upto = mine;
        for (int o = 1; o < 64; o <<= 1) {
            const double y = __shfl_up(upto, o);
            if (lane >= o) upto += y;
        }
        if (lane == 63) ends[wave] = upto;
        __syncthreads();
        double total = 0.0, before = 0.0;
        for (int v = 0; v < kVerifyWaves; ++v) {
            if (v < wave) before += ends[v];
            total += ends[v];
        }
        chunk[t] = before + upto;
        if (t == 0) {
            lds_tile = -1;
            lds_first = kVerifyThreads;
            lds_total = total;
        }
        __syncthreads();
        if (lds_total > 0.0) break;
        // nothing is left of p - q (a u of 1, no number): of p itself
        w.draft = false;
        w.one = -1;
        verify_sums<DT>(a, pl, w, b, n, wave, kVerifyWaves);
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
    }
    const double border = u * lds_total;
    // the first thread whose run ends above the border; rounding may leave none:
    // then the last one that adds anything
    if (first < end && chunk[t] > border) atomicMin(&lds_first, t);
    __syncthreads();
    if (t == lds_first) {
        double sum = t ? chunk[t - 1] : 0.0;
        int at = end - 1;
        double start = sum;
        for (int i = first; i < end; ++i) {
            start = sum;
            sum += ld_device(sums + i);
            if (sum > border) {
                at = i;
                break;
            }
        }
        lds_tile = at;
        lds_before = start;
    }
    __syncthreads();
    if (wave == 0) {
        int tile = lds_tile;
        double sum = lds_before;
        const bool past = tile < 0;
        if (past) {  // (the last tile that holds anything)
            int at = -1;
            for (int i = lane; i < pl.tiles; i += 64)
                if (ld_device(sums + i) > 0.0) at = i;
            tile = max(0, -wave_least(-at));
            sum = 0.0;
        }
        const int base = tile * kVerifyTile;
        R p, q;
        p.load(verify_row<T>(a, b, n), base, a.V);
        if (w.draft) q.load(verify_row<T>(a, b, a.T + 1 + n), base, a.V);
        double left[kVerifyPer];
        verify_left<DT>(w, p, q, base, left);
        int token = -1, last = -1;  // the first above the border; the last that is left at all
#pragma unroll
        for (int v = 0; v < R::NV; ++v) {
            double s = 0.0;
#pragma unroll
            for (int i = 0; i < R::W; ++i) {
                s += left[v * R::W + i];
                if (left[v * R::W + i] > 0.0) last = R::index(base, v * R::W + i);
            }
            double upto = s;
            for (int o = 1; o < 64; o <<= 1) {
                const double y = __shfl_up(upto, o);
                if (lane >= o) upto += y;
            }
            double run = __shfl_up(upto, 1);
            run = sum + (lane ? run : 0.0);
            if (!past && token < 0) {
                const uint64_t above = __ballot(sum + upto > border);
                if (above) {
                    const int l = __builtin_ctzll(above);
                    int at = -1;
#pragma unroll
                    for (int i = 0; i < R::W; ++i) {
                        run += left[v * R::W + i];
                        const bool over = run > border || i == R::W - 1;
                        if (at < 0 && over && left[v * R::W + i] > 0.0) at = R::index(base, v * R::W + i);
                    }
                    // (rounding: the lane's last that is left)
                    if (at < 0)
                        for (int i = 0; i < R::W; ++i)
                            if (left[v * R::W + i] > 0.0) at = R::index(base, v * R::W + i);
                    token = __shfl(at, l);
                }
            }
            sum += __shfl(upto, 63);
        }
        last = -wave_least(-last);
        if (token < 0) token = last < 0 ? 0 : last;
        if (lane == 0) lds_tile = token;
    }
    __syncthreads();
    finish(lds_tile);
}

namespace {

VerifyPlan make_plan(const VerifyArgs& a, int cus) {
    VerifyPlan pl;
    pl.rows = a.T + 1 + (a.draft ? a.T : 0);
    pl.tiles = (a.V + kVerifyTile - 1) / kVerifyTile;
    const int64_t rows = (int64_t)a.S * pl.rows, most = (pl.tiles + kVerifyWaves - 1) / kVerifyWaves;
    const int64_t want = std::max<int64_t>(1, 8 * (int64_t)cus / rows);
    pl.slices = (int)std::min<int64_t>(std::min<int64_t>(want, kVerifySlices), most);
    const int per = (pl.tiles + pl.slices - 1) / pl.slices;
    pl.slices = (pl.tiles + per - 1) / per;
    pl.blocks = (int)std::min<int64_t>(most, std::max<int64_t>(1, 4 * (int64_t)cus / a.S));
    pl.stats = nullptr;
    pl.sums = nullptr;
    pl.count = nullptr;
    return pl;
}

template <int DT>
hipError_t launch(const VerifyArgs& a, const VerifyPlan& pl, hipStream_t s) {
    verify_stats_kernel<DT><<<(unsigned)((int64_t)a.S * pl.rows * pl.slices), kVerifyThreads, 0, s>>>(a, pl);
    if (const hipError_t e = hipGetLastError(); e != hipSuccess) return e;
    verify_draw_kernel<DT><<<(unsigned)((int64_t)a.S * pl.blocks), kVerifyThreads, 0, s>>>(a, pl);
    return hipGetLastError();
}

}  // namespace

size_t verify_workspace(const VerifyArgs& a, int cus, size_t* counters) {
    const VerifyPlan pl = make_plan(a, cus);
    *counters = (size_t)a.S * sizeof(unsigned);
    return (size_t)a.S * pl.rows * pl.slices * sizeof(RowStat) + (size_t)a.S * pl.tiles * sizeof(double);
}

hipError_t launch_verify(int dtype, const VerifyArgs& a, int cus, void* ws, void* counters, hipStream_t s) {
    VerifyPlan pl = make_plan(a, cus);
    pl.stats = static_cast<RowStat*>(ws);
    pl.sums = reinterpret_cast<double*>(pl.stats + (size_t)a.S * pl.rows * pl.slices);
    pl.count = static_cast<unsigned*>(counters);
    switch (dtype) {
        case XT_F32: return launch<XT_F32>(a, pl, s);
        case XT_F16: return launch<XT_F16>(a, pl, s);
        default: return launch<XT_BF16>(a, pl, s);
    }
}

}  // namespace xt
