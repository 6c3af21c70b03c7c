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
// p and q are e / l, e = exp((x - m) / temperature) and l the sum of a row's; both
// sides of a comparison are multiplied by the rows' l instead: u e_q l_p < e_p l_q,
// and what is left in units of 1 / (l_p l_q), or 1 / l_p.  Equal logits have e = 1 to
// the bit, so that their sums are whole numbers and a border that lies on one is
// met exactly.
//
// Everything that decides is in 64 bits: a token flips where a sum of V terms
// crosses a border, and f32 exponentials would move some of V borders by 1e-8
// each.  The first kernel reads every row that can count once (HBM bounds large
// calls: f64 instructions go at the rate of f32 ones), rows cut into slices
// where they are few; the second decides, reads the one row that is drawn from
// again, in tiles of 512 logits a wave, and the workgroup that ends the
// sequence's last tile finds the tile and in it the token (sums and count at
// device scope, as the chip's eight L2s need it).
// 64 sequences of 4 drafts, 128003 bf16 logits: 53 + 30.5 us, where HBM would take 23:
// 22 f64 instructions a logit are 36 us of the first kernel.  One sequence of 128256
// f32 logits: 5.6 + 13.1 us, the second one a chain of eight dependent trips to
// memory (sums, drafts, their logits, the row, stores, count, tile sums, the tile).
#include <algorithm>

#include "xtern_cache.h"

namespace xt {

constexpr int kVerifyThreads = 256;
constexpr int kVerifyWaves = kVerifyThreads / 64;
constexpr int kStatsPer = 16;                      // logits of a lane and tile, in the first kernel
constexpr int kDrawPer = 8;                        // and in the second
constexpr int kStatsTile = 64 * kStatsPer;         // of a wave
constexpr int kDrawTile = 64 * kDrawPer;
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
    double* sums;     // [S][draws]
    unsigned* count;  // [S]: workgroups done, zero between calls
    int rows;         // of a sequence: T + 1, and T of the draft
    int slices, tiles, per;  // of a row, in the first kernel; tiles of a slice
    int draws, blocks;       // tiles of a row in the second kernel, workgroups of a sequence
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

// 2^y for y <= 0: y = n + f, |f| <= 1/2, a polynomial of 2^f of degree 9 through
// its values in Chebyshev's nodes (the constant term then made 1, so that 0 gives
// 1), 3e-14 of the result, and n added to its exponent.  n: the last bits of *z.
__device__ __forceinline__ double verify_pow2(double y, double* z) {
    const double magic = 0x1.8p52;
    *z = y + magic;
    const double f = y - (*z - magic);
    double p = 0x1.b6571de2f2351p-24;
    p = fma(p, f, 0x1.63ef969a64d3cp-20);
    p = fma(p, f, 0x1.ffcb76789860fp-17);
    p = fma(p, f, 0x1.43088e257f341p-13);
    p = fma(p, f, 0x1.5d87fe908f88ap-10);
    p = fma(p, f, 0x1.3b2ab72b175eep-7);
    p = fma(p, f, 0x1.c6b08d7044119p-5);
    p = fma(p, f, 0x1.ebfbdff8149f2p-3);
    p = fma(p, f, 0x1.62e42fefa39f7p-1);
    return fma(p, f, 1.0);
}
// exp((x - m) / temperature) for x <= m, c = log2 e / temperature; 0 for x =
// -inf; the caller sees to NaN and +inf.
__device__ __forceinline__ double verify_exp(float x, float m, double c) {
    double z;
    const double p = verify_pow2(fmax(((double)x - (double)m) * c, -1100.0), &z);
    return ldexp(p, (int)__builtin_bit_cast(int64_t, z));
}
// The same for a sum of at least 1: 2^-1000 instead of anything less.  (m itself
// gives 1 to the last bit here as well: where p and q have nearly all of it on one
// token, what is left is the difference of two numbers next to 1.)
__device__ __forceinline__ double verify_term(float x, double m, double c) {
    double z;
    const double p = verify_pow2(fmax(((double)x - m) * c, -1000.0), &z);
    const uint64_t bits = __builtin_bit_cast(uint64_t, p);
    const unsigned hi = (unsigned)(bits >> 32) + ((unsigned)__builtin_bit_cast(uint64_t, z) << 20);
    return __builtin_bit_cast(double, ((uint64_t)hi << 32) | (unsigned)bits);
}
__device__ __forceinline__ double verify_rate(float temp) {
    return temp > 0.0f ? 1.4426950408889634 / (double)temp : 0.0;
}

// A lane's logits of a tile: vectors of 16 bytes (W logits), vector v at base +
// (v * 64 + lane) * W; -inf past the row.
template <int DT, int PER>
struct VerifyTile {
    static constexpr int W = DT == XT_F32 ? 4 : 8, NV = PER / W;
    typedef typename Elem<DT>::T T;
    typedef T Vec __attribute__((ext_vector_type(W)));
    typedef Vec VecU __attribute__((aligned(sizeof(T))));
    float x[PER];
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

// Over the wave, in every lane.
__device__ __forceinline__ double wave_add(double v) { return lanes_sum<64>(v); }
template <typename Op>
__device__ __forceinline__ int wave_of(int v, Op op) {
    v = op(v, dpp_to<0xb1>(v));
    v = op(v, dpp_to<0x4e>(v));
    v = op(v, dpp_to<0x141>(v));
    v = op(v, dpp_to<0x140>(v));
    auto a = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = op((int)a[0], (int)a[1]);
    auto b = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return op((int)b[0], (int)b[1]);
}
__device__ __forceinline__ float wave_most(float v) {
    return __int_as_float(wave_of(__float_as_int(v), [](int a, int b) {
        return __float_as_int(fmaxf(__int_as_float(a), __int_as_float(b)));
    }));
}
__device__ __forceinline__ int wave_least(int v) {
    return wave_of(v, [](int a, int b) { return min(a, b); });
}
// Inclusive sums over the lanes.
template <int CTRL, int ROWS>
__device__ __forceinline__ double dpp_add(double v) {
    return v + __hiloint2double(dpp_id<CTRL, ROWS>(__double2hiint(v)), dpp_id<CTRL, ROWS>(__double2loint(v)));
}
__device__ __forceinline__ double wave_upto(double v) {
    v = dpp_add<0x111, 0xf>(v);
    v = dpp_add<0x112, 0xf>(v);
    v = dpp_add<0x114, 0xf>(v);
    v = dpp_add<0x118, 0xf>(v);
    v = dpp_add<0x142, 0xa>(v);
    return dpp_add<0x143, 0xc>(v);
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
    typedef VerifyTile<DT, kStatsPer> R;
    __shared__ RowStat waves[kVerifyWaves];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int slice = blockIdx.x % pl.slices, row = blockIdx.x / pl.slices, b = row / pl.rows, j = row % pl.rows;
    const int count = verify_count(a, b);
    if (j <= a.T ? j > count : j - a.T - 1 >= count) return;
    const float temp = verify_temp(a, b);
    const double c = verify_rate(temp);
    const typename R::T* x = verify_row<typename R::T>(a, b, j);
    const int per = pl.per, t1 = min(pl.tiles, (slice + 1) * per);
    RowStat s{0.0, -INFINITY, 0x7fffffff};
    bool bad = false;
    for (int t = slice * per + wave; t < t1; t += kVerifyWaves) {
        R r;
        r.load(x, t * kStatsTile, a.V);
        float m = r.x[0];
#pragma unroll
        for (int i = 1; i < kStatsPer; ++i) m = __builtin_elementwise_maximum(m, r.x[i]);  // (NaN stays)
        bad |= !(m < INFINITY);
        if (temp > 0.0f) {
            if (m > s.m) {
                s.l *= s.m == -INFINITY ? 0.0 : verify_exp(s.m, m, c);
                s.m = m;
            }
            if (s.m == -INFINITY) continue;  // (nothing yet)
            const double base = s.m;
            // (two sums: half the chain)
            double l0 = 0.0, l1 = 0.0;
#pragma unroll
            for (int i = 0; i < kStatsPer; i += 2) {
                l0 += verify_term(r.x[i], base, c);
                l1 += verify_term(r.x[i + 1], base, c);
            }
            s.l += l0 + l1;
        } else if (m > s.m) {
            int at = 0x7fffffff;
#pragma unroll
            for (int i = kStatsPer - 1; i >= 0; --i)
                if (r.x[i] == m) at = R::index(t * kStatsTile, i);
            s.m = m;
            s.at = at;
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

// What the second kernel draws from: max(p - q, 0) in units of 1 / (l_p l_q); without
// draft logits p, or p without one token, in units of 1 / l_p.
struct VerifyDraw {
    float pm, qm;
    double pl, ql;  // the factors of exp((x - m) / temperature): the other row's l; 1
    double c;
    int one;        // all of q: this token (draft NULL), -1: none of it
    bool draft;     // q of the draft's logits
};
__device__ __forceinline__ double verify_left(const VerifyDraw& w, float x, float y, int at) {
    double v = verify_exp(x, w.pm, w.c) * w.pl;
    if (w.draft) v = fmax(v - verify_exp(y, w.qm, w.c) * w.ql, 0.0);
    return at == w.one ? 0.0 : v;
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
    typedef VerifyTile<DT, kDrawPer> R;
    const typename R::T* prow = verify_row<typename R::T>(a, b, n);
    const typename R::T* qrow = w.draft ? verify_row<typename R::T>(a, b, a.T + 1 + n) : prow;
    for (int t = first; t < pl.draws; t += step) {
        R p, q;
        p.load(prow, t * kDrawTile, a.V);
        if (w.draft) q.load(qrow, t * kDrawTile, a.V);
        double sum = 0.0;
#pragma unroll
        for (int i = 0; i < kDrawPer; ++i) sum += verify_left(w, p.x[i], q.x[i], R::index(t * kDrawTile, i));
        sum = wave_add(sum);
        if ((threadIdx.x & 63) == 0) st_device(pl.sums + (int64_t)b * pl.draws + t, sum);
    }
}

template <int DT>
__global__ __launch_bounds__(kVerifyThreads) void verify_draw_kernel(VerifyArgs a, VerifyPlan pl) {
    typedef VerifyTile<DT, kDrawPer> R;
    typedef typename R::T T;
    __shared__ RowStat rows[kVerifyRows];
    __shared__ double ends[kVerifyWaves];
    __shared__ int lds_n, lds_x, lds_last, lds_tile, lds_first;
    __shared__ double lds_before;
    const int b = blockIdx.x / pl.blocks, block = blockIdx.x % pl.blocks;
    const int t = threadIdx.x, wave = t >> 6, lane = t & 63;
    const int count = verify_count(a, b);
    const float temp = verify_temp(a, b);
    const double c = verify_rate(temp);
    const bool there = count >= 0 && temp >= 0.0f && temp < INFINITY;
    const double share = a.uniforms[(int64_t)b * (a.T + 1) + a.T];
    // (wave 0) lane t: draft t, its logits and its number, on their way while the
    // rows' sums are joined.  Neither waits for the count: drafts and sums behind it
    // are read and not used (13.1 us of kernel for one sequence, 13.8 before)
    int id = -1;
    float u = 0.0f, px = 0.0f, qx = 0.0f;
    if (wave == 0 && lane < a.T) {
        id = a.drafted[(int64_t)b * a.T + lane];
        u = a.uniforms[(int64_t)b * (a.T + 1) + lane];
        if ((unsigned)id < (unsigned)a.V) {
            px = Elem<DT>::get(verify_row<T>(a, b, lane)[id]);
            if (a.draft) qx = Elem<DT>::get(verify_row<T>(a, b, a.T + 1 + lane)[id]);
        }
    }
    // the rows' sums, four rows of a wave at a time
    for (int j0 = wave; j0 < pl.rows; j0 += 4 * kVerifyWaves) {
        RowStat s[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int j = j0 + i * kVerifyWaves;
            s[i] = RowStat{0.0, -INFINITY, 0x7fffffff};
            if (lane < pl.slices && j < pl.rows)
                s[i] = pl.stats[((int64_t)b * pl.rows + j) * pl.slices + lane];
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int j = j0 + i * kVerifyWaves;
            if (j >= pl.rows) break;
            s[i] = wave_join(s[i], c);
            if (temp == 0.0f) s[i].l = s[i].m == -INFINITY ? NAN : s[i].l + 1.0;
            if (lane == 0) rows[j] = s[i];
        }
    }
    __syncthreads();
    // a row of probabilities: its sum is a number, and not 0
    auto fine = [&](int j) { return rows[j].l > 0.0 && rows[j].l < INFINITY; };
    auto term = [&](int j, float x) { return verify_exp(x, rows[j].m, c); };
    if (wave == 0) {
        // whether the draft is accepted
        const bool mine = there && lane < count;
        if (!mine) id = -1;
        bool taken = false;
        if (mine && (unsigned)id < (unsigned)a.V && fine(lane) && (!a.draft || fine(a.T + 1 + lane))) {
            if (temp == 0.0f)
                taken = id == rows[lane].at;
            else if (a.draft)
                taken = (double)u * term(a.T + 1 + lane, qx) * rows[lane].l < term(lane, px) * rows[a.T + 1 + lane].l;
            else
                taken = (double)u * rows[lane].l < term(lane, px);
        }
        const uint64_t no = ~__ballot(taken);
        const int accepted = there ? min(no ? (int)__builtin_ctzll(no) : 64, count) : 0;
        if (lane == accepted) lds_x = id;
        if (lane == 0) lds_n = accepted;
        if (lane == 0 && accepted == 64) lds_x = -1;
    }
    __syncthreads();
    const int n = lds_n;
    // the draft that was not accepted; none, or one that is no token: all of p is left
    const int x = lds_x;
    const bool refused = (unsigned)x < (unsigned)a.V;
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
    w.c = c;
    w.draft = refused && a.draft;
    w.one = refused && !a.draft ? x : -1;
    w.pl = w.draft ? rows[a.T + 1 + n].l : 1.0;
    w.qm = w.draft ? rows[a.T + 1 + n].m : 0.0f;
    w.ql = w.draft ? rows[n].l : 0.0;
    verify_sums<DT>(a, pl, w, b, n, block * kVerifyWaves + wave, pl.blocks * kVerifyWaves);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // every store has arrived
    __syncthreads();
    // (the count wraps to zero by itself, for the next call)
    if (t == 0) lds_last = atomicInc(pl.count + b, (unsigned)pl.blocks - 1) == (unsigned)pl.blocks - 1;
    __syncthreads();
    if (!lds_last) return;
    // Sums over the workgroup's threads before each, and of all.
    auto scan = [&](double v, double* total) {
        const double upto = wave_upto(v), before = __shfl_up(upto, 1);
        if (lane == 63) ends[wave] = upto;
        if (t == 0) lds_first = kVerifyThreads;
        __syncthreads();
        double first = lane ? before : 0.0;
        *total = 0.0;
        for (int i = 0; i < kVerifyWaves; ++i) {
            if (i < wave) first += ends[i];
            *total += ends[i];
        }
        return first;
    };
    // The tile: a run of tiles a thread
    const int per = (pl.draws + kVerifyThreads - 1) / kVerifyThreads, first = t * per, end = min(pl.draws, first + per);
    const double* sums = pl.sums + (int64_t)b * pl.draws;
    double before, total, run, four[4];  // (four of the run's tiles on their way)
    auto fetch = [&](int i0) {
#pragma unroll
        for (int i = 0; i < 4; ++i) four[i] = ld_device(sums + min(i0 + i, pl.draws - 1));
    };
    for (int pass = 0;; ++pass) {
        run = 0.0;
        for (int i0 = first; i0 < end; i0 += 4) {
            fetch(i0);
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (i0 + i < end) run += four[i];
        }
        before = scan(run, &total);
        if (total > 0.0 || pass) break;
        // nothing is left of p - q (a u of 1, no number): of p itself
        w.draft = false;
        w.one = -1;
        w.pl = 1.0;
        verify_sums<DT>(a, pl, w, b, n, wave, kVerifyWaves);
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
    }
    const double border = share < 1.0 ? share * total : INFINITY;
    // The first thread whose run adds anything and ends above the border, in it the
    // first such tile; rounding may leave none: then the last one that adds
    // anything.  (The sums before two threads are rounded in different orders, so a
    // border on a sum may be passed between them, by a run of nothing but 0.)
    if (run > 0.0 && before + run > border) atomicMin(&lds_first, t);
    if (t == 0) lds_tile = -1;
    __syncthreads();
    const bool past = lds_first == kVerifyThreads;
    if (t == lds_first) {
        double sum = before;
        int at = per > 1 ? -1 : first;
        lds_before = sum;
        for (int i0 = first; i0 < end && per > 1; i0 += 4) {
            if (per > 4) fetch(i0);
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (i0 + i < end && four[i] > 0.0 && (at < 0 || sum <= border)) {
                    lds_before = sum;
                    sum += four[i];
                    at = i0 + i;
                }
            if (at >= 0 && sum > border) break;
        }
        lds_tile = at;
    } else if (past) {
        for (int i = first; i < end; ++i)
            if (ld_device(sums + i) > 0.0) atomicMax(&lds_tile, i);
    }
    __syncthreads();
    // The token: kEach of the tile's logits a thread
    constexpr int kEach = kDrawTile / kVerifyThreads;
    const int at = max(lds_tile, 0) * kDrawTile + t * kEach;
    const T* prow = verify_row<T>(a, b, n);
    const T* qrow = w.draft ? verify_row<T>(a, b, a.T + 1 + n) : prow;
    double left[kEach], mine_left = 0.0;
    int last = -1;  // the last that is left at all
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
        left[i] = at + i < a.V ? verify_left(w, Elem<DT>::get(prow[at + i]), Elem<DT>::get(qrow[at + i]), at + i) : 0.0;
        mine_left += left[i];
        if (left[i] > 0.0) last = at + i;
    }
    double sum = past ? 0.0 : lds_before;
    sum += scan(mine_left, &total);
    if (!past && last >= 0 && sum + mine_left > border) atomicMin(&lds_first, t);
    if (t == 0) lds_x = 0;
    __syncthreads();
    if (t == lds_first) {
        int token = last;
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            sum += left[i];
            if (sum > border && left[i] > 0.0) {
                token = at + i;
                break;
            }
        }
        lds_x = token;
    } else if (lds_first == kVerifyThreads && last >= 0) {
        atomicMax(&lds_x, last);
    }
    __syncthreads();
    finish(lds_x);
}

namespace {

VerifyPlan make_plan(const VerifyArgs& a, int cus) {
    VerifyPlan pl;
    pl.rows = a.T + 1 + (a.draft ? a.T : 0);
    pl.tiles = (a.V + kStatsTile - 1) / kStatsTile;
    pl.draws = (a.V + kDrawTile - 1) / kDrawTile;
    const int64_t rows = (int64_t)a.S * pl.rows, most = (pl.tiles + kVerifyWaves - 1) / kVerifyWaves;
    // Slices, of a tile a wave at least, until 32 workgroups per compute unit: four
    // times as many as run at once, for the rows behind a sequence's drafts end at
    // once (until 12 / 20 / 32: 64 sequences of 4 drafts 60 / 54 / 53 us)
    const int64_t want = std::max<int64_t>(1, 32 * (int64_t)cus / rows);
    pl.slices = (int)std::min<int64_t>(std::min<int64_t>(want, kVerifySlices), most);
    pl.per = (int)((most + pl.slices - 1) / pl.slices) * kVerifyWaves;
    pl.slices = (pl.tiles + pl.per - 1) / pl.per;
    // Workgroups of a sequence, until two per compute unit (one / two / four: 13
    // sequences without drafts of 192299 logits 23.6 / 23.8 / 28.7 us for both
    // kernels, 64 of 4 drafts and 128003 91.4 / 86.3 / 86.0)
    pl.blocks = (int)std::min<int64_t>((pl.draws + kVerifyWaves - 1) / kVerifyWaves,
                                       std::max<int64_t>(1, 2 * (int64_t)cus / a.S));
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
    return (size_t)a.S * pl.rows * pl.slices * sizeof(RowStat) + (size_t)a.S * pl.draws * sizeof(double);
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
