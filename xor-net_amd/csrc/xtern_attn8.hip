// Attention over a paged cache of 8-bit codes with a scale for each position
// and key-value head.
#include "xtern_attn.h"

namespace xt {

// For each row and query head, over the positions j that the row sees and whose
// page exists, with key codes kc, value codes vc and their scales ks, vs:
// s_j = scale ks_j (q . kc_j), m = max s, l = sum exp(s_j - m),
// out = sum (exp(s_j - m) vs_j) vc_j / l, lse = m + ln l.
//
// The cache is read once, so HBM bounds it: a position of one key-value head is
// 2 D + 8 bytes.  The products run on the 8-bit matrix cores as they are, the
// codes never become floats: an f32 operand x (a query, or the 16 columns'
// weights exp(s - m) vs) is rounded to a whole number of 24 bits, x 2^k, with
// the largest of its column near 2^23, and that to three signed 8-bit digits,
// whose products with the codes add up in 32-bit integers without rounding.
// What is lost is half a unit of the column's largest operand, which is 4177856
// or more: of the query once, of the weights in each tile of 64 positions on its
// own.
// The columns are the query heads of a group, and the groups of several rows
// where rows share a sequence (16 / group rows): drafts and prompts read the
// cache once for all of these.  As in the 16-bit kernel everything is
// transposed: S^T = K Q^T gives a lane four positions of its own column per 16,
// which are its operand of O^T = V^T P^T; the value rows it loads as pieces and
// transposes in registers (v_perm), and only a column's maximum crosses lanes.
// At D = 128 a tile of 64 positions is 16.9 KB, 48 matrix instructions of 16 cycles
// and about 390 others, which take the chip half of the time that HBM takes.
// 32 and 8 heads of 128: 131072 positions 56 us (4.9 TB/s), 64 rows of up to 8192
// 101 to 107 (5.2 to 5.5); 700 positions of 20 and 5 heads 13 us, 32 positions 10:
// the chain of dependent loads (lengths, table, scales and codes, the join's).
// Value rows are read with the streaming hint (without: 57 and 124 us), key rows
// are not, whose lines several loads read (with: 61 and 117).

// (rows may start at any byte)
typedef v4i v4ib __attribute__((aligned(1)));
typedef v2i v2ib __attribute__((aligned(1)));
typedef int v1ib __attribute__((aligned(1)));

template <int DP>
struct Attn8Shape {
    static constexpr int TK = 64;       // positions per tile of a wave
    static constexpr int NT = TK / 16;
    static constexpr int KS = DP / 64;  // key loads per 16 positions
    static constexpr int NJ = TK / 4;   // positions of a lane's V piece
    static constexpr int UE = DP / 16;  // elements of a value load
};
constexpr int kDigits = 3;
constexpr float kMostDigits = 8355711.0f;  // 0x7f7f7f
// Value scales that the digits' exponents have no room for go the plain way.
constexpr float kLeastScale = 0x1p-90f;

// k such that x 2^k, x the largest of a column, is a number of three digits and
// not one of 22 bits; the digits of whole numbers in the bytes 0 .. 2.
__device__ __forceinline__ int digit_shift(float x) {
    const int k = 23 - __builtin_amdgcn_frexp_expf(x);
    return min(126, ldexpf(x, k) > kMostDigits ? k - 1 : k);
}
__device__ __forceinline__ unsigned digits_of(int v) { return ((unsigned)v + 0x808080u) ^ 0x808080u; }

// Four numbers' digits -> a dword of each digit.
__device__ __forceinline__ void gather_digits(const unsigned* x, int* out) {
    const unsigned a = __builtin_amdgcn_perm(x[1], x[0], 0x05010400u), b = __builtin_amdgcn_perm(x[3], x[2], 0x05010400u);
    const unsigned c = __builtin_amdgcn_perm(x[1], x[0], 0x0c0c0602u), d = __builtin_amdgcn_perm(x[3], x[2], 0x0c0c0602u);
    out[0] = (int)__builtin_amdgcn_perm(b, a, 0x05040100u);
    out[1] = (int)__builtin_amdgcn_perm(b, a, 0x07060302u);
    out[2] = (int)__builtin_amdgcn_perm(d, c, 0x05040100u);
}

// Four rows of four bytes -> four columns of four.
__device__ __forceinline__ void transpose4(const int* x, int* out) {
    const unsigned a = __builtin_amdgcn_perm(x[1], x[0], 0x05010400u), b = __builtin_amdgcn_perm(x[3], x[2], 0x05010400u);
    const unsigned c = __builtin_amdgcn_perm(x[1], x[0], 0x07030602u), d = __builtin_amdgcn_perm(x[3], x[2], 0x07030602u);
    out[0] = (int)__builtin_amdgcn_perm(b, a, 0x05040100u);
    out[1] = (int)__builtin_amdgcn_perm(b, a, 0x07060302u);
    out[2] = (int)__builtin_amdgcn_perm(d, c, 0x05040100u);
    out[3] = (int)__builtin_amdgcn_perm(d, c, 0x07060302u);
}

// A workgroup's columns: heads h0 .. of one row, or the group's heads of
// several.
struct Attn8Cols {
    int row, h0, G, n;
    FastDiv by_group;
    bool several;
    __device__ __forceinline__ AttnPlace operator()(int x) const {
        if (!several) return AttnPlace{row, h0 + x};
        const int t = fast_quot(x, by_group);
        return AttnPlace{row + t, h0 + x - t * G};
    }
};

struct Attn8Call {
    AttnArgs a;
    AttnPlan pl;
    float scale2;
    int G;  // query heads of a group
    FastDiv by_group, by_tiles;
};

// Whether a row of length n sees position p.
__device__ __forceinline__ bool attn_sees(const AttnArgs& a, int n, int p) {
    return (p < n) & ((p < a.sink) | (p >= n - a.window));
}

// One chunk of a unit in plain f32 operations: queries and scales that are
// infinite, NaN or beyond the digits' exponents, and head sizes below one load.
// 256 positions at a time, one column after the other.
__device__ void attn8_plain(const AttnArgs& a, const AttnSeg& it, int hk, const Attn8Cols& cols,
                            float scale2, float* lds_o, float* lds_ml, int ldo) {
    const KvView& c = a.c;
    const int t = threadIdx.x;
    __shared__ float sp[kAttnThreads], sv[kAttnThreads];
    __shared__ int64_t so[kAttnThreads];
    __shared__ float sm[kAttnWaves];
    const int8_t* kc = static_cast<const int8_t*>(c.k);
    const int8_t* vc = static_cast<const int8_t*>(c.v);
    for (int x = 0; x < cols.n; ++x) {
        const AttnPlace w = cols(x);
        const int len = kv_length(c, a.lengths[w.row]);
        const float* q = a.q + w.row * a.ldq + (int64_t)w.head * c.D;
        float m = -INFINITY, l = 0.0f, o = 0.0f;
        for (int p0 = it.p0; p0 < it.p1; p0 += kAttnThreads) {
            const int p = attn_pos<true>(a, it.gap, p0 + t);
            const int pg = p0 + t < it.p1 && attn_sees(a, len, p) ? kv_page(c, it.seq, p) : -1;
            const int64_t off = pg < 0 ? -1 : kv_offset(c, pg, p, hk);
            float s = -INFINITY, vs = 0.0f;
            if (off >= 0) {
                const int64_t at = ((int64_t)pg * c.hkv + hk) * c.page + kv_slot(c, p);
                const float ks = a.ks[at];
                vs = a.vs[at];
                float acc = 0.0f;
                for (int d = 0; d < c.D; ++d) acc += q[d] * (ks * (float)kc[off + d]);
                s = acc * scale2;
            }
            float v = s;
            for (int y = 32; y; y >>= 1) v = fmaxf(v, __shfl_xor(v, y));
            __syncthreads();
            if ((t & 63) == 0) sm[t >> 6] = v;
            so[t] = off;
            sv[t] = vs;
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
                    if (t < c.D) o += sp[j] * (sv[j] * (float)vc[so[j] + t]);
                }
            __syncthreads();
        }
        if (t < c.D) lds_o[x * ldo + t] = o;
        if (t == 0) {
            lds_ml[x] = m;
            lds_ml[16 + x] = l;
        }
    }
    __syncthreads();
}

// Four elements of a column's sums: into its row's result, divided by l; into
// a segment's.
__device__ __forceinline__ void attn8_out(const AttnArgs& a, AttnPlace w, int d, v4f sum, float l) {
    const int D = a.c.D;
    float* to = a.out + w.row * a.ldo + (int64_t)w.head * D + d;
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    sum *= inv;
    if (l == 0.0f) sum = v4f{0.0f, 0.0f, 0.0f, 0.0f};
    if (d + 4 <= D) {
        *reinterpret_cast<v4fu*>(to) = sum;
    } else {
#pragma unroll
        for (int e = 0; e < 3; ++e)
            if (d + e < D) to[e] = sum[e];
    }
}
__device__ __forceinline__ void attn8_part(const AttnPlan& pl, int64_t item, int h, int d, int D, v4f sum) {
    float* to = pl.part_o + (item * 16 + h) * pl.dp + d;
    st2_device(to, sum[0], d + 1 < D ? sum[1] : 0.0f);
    if (d + 2 < D) st2_device(to + 2, sum[2], d + 3 < D ? sum[3] : 0.0f);
}

// Joins `cnt` (at most 64) segments, in every `every`-th slot from slot0, of all
// columns: into the rows' results (last), or into slot0.  As at the end of a
// segment a thread has four elements of a column; where columns are few, 2, 4 or
// 8 threads share them, each every 2nd, 4th or 8th segment.  Bound by the latency
// of device-scope loads: up to 16 segments of a thread are on their way at once,
// while the segments' statistics go through LDS (scratch, 4096 floats).
template <int DP>
__device__ void attn8_join(const AttnArgs& a, const AttnPlan& pl, const Attn8Cols& cols, int tid, int heads,
                           int64_t slot0, int every, int cnt, bool last, float* scratch) {
    constexpr int N = DP == 64 ? 8 : 16, Q = DP / 4;  // segments in flight (as registers allow), threads of a column
    const int D = a.c.D;
    const int64_t first = slot0 * pl.hy + heads, step = (int64_t)every * pl.hy;
    float2* stats = reinterpret_cast<float2*>(scratch);      // [cnt][16]
    v4f* sums = reinterpret_cast<v4f*>(scratch + 64 * 16 * 2);  // [256]
    // columns that are worked on at once, rounded up to a power of two
    const int lg = cols.n > 1 ? 32 - __builtin_clz(cols.n - 1) : 0;
    const int wide = min(Q << lg, kAttnThreads), parts = kAttnThreads / wide;
    const int part = tid / wide, x = tid & (wide - 1), d = x % Q * 4;
    float2 st[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int e = tid + kAttnThreads * i;
        if (e < 16 * cnt && e % 16 < cols.n) st[i] = ld2_device(pl.part_ml + ((first + e / 16 * step) * 16 + e % 16) * 2);
    }
#pragma unroll 1
    for (int h0 = 0; h0 < cols.n; h0 += wide / Q) {
        const int h = min(h0 + x / Q, cols.n - 1);
        const bool in = h0 + x / Q < cols.n && d < D;
        const float* from = pl.part_o + (first * 16 + h) * pl.dp + min(d, pl.dp - 2);
        const int more = d + 2 < pl.dp ? 2 : 0;
        const int64_t stride = step * 16 * pl.dp;
        float m = -INFINITY, l = 0.0f;
        v4f sum = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 1
        for (int c0 = 0; c0 < cnt; c0 += N * parts) {
            float2 lo[N], hi[N];
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int c = c0 + i * parts + part;
                if (c0 + i * parts < cnt) {  // (the same for all threads)
                    const float* y = from + min(c, cnt - 1) * stride;
                    lo[i] = ld2_device(y);
                    hi[i] = ld2_device(y + more);
                }
            }
            if (c0 == 0) {
                if (h0 == 0) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int e = tid + kAttnThreads * i;
                        if (e < 16 * cnt && e % 16 < cols.n) stats[e] = st[i];
                    }
                    __syncthreads();
                }
                for (int c = 0; c < cnt; ++c) m = fmaxf(m, stats[16 * c + h].x);
            }
            const float base = m == -INFINITY ? 0.0f : m;
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int c = c0 + i * parts + part;
                if (c0 + i * parts < cnt) {
                    const float2 s = stats[16 * min(c, cnt - 1) + h];
                    const float f = c < cnt ? pow2(s.x - base) : 0.0f;
                    l += s.y * f;
                    if (c < cnt) sum += f * v4f{lo[i].x, lo[i].y, hi[i].x, hi[i].y};
                }
            }
        }
        if (parts > 1) {  // (then the columns are all here)
            float* ls = reinterpret_cast<float*>(sums + kAttnThreads);
            sums[tid] = sum;
            ls[tid] = l;
            __syncthreads();
            for (int p = 1; p < parts && part == 0; ++p) {
                sum += sums[tid + p * wide];
                l += ls[tid + p * wide];
            }
        }
        if (!in || part) continue;
        if (last) attn8_out(a, cols(h), d, sum, l);
        else attn8_part(pl, first, h, d, D, sum);  // (what lay there has been read)
        if (d) continue;
        if (!last) {
            st2_device(pl.part_ml + (first * 16 + h) * 2, m, l);
        } else if (a.lse) {
            const AttnPlace w = cols(h);
            a.lse[(int64_t)w.row * a.hq + w.head] = row_lse(m, l);
        }
    }
}

template <int DP>
__global__ __launch_bounds__(kAttnThreads, DP == 256 ? 1 : (DP == 128 ? 2 : 3)) void attention8_kernel(Attn8Call call) {
    typedef Attn8Shape<DP> S;
    constexpr int kLdsRow = DP + 4;  // floats; the pad keeps columns apart in the banks
    constexpr int kItems = 16 * DP / 4 / kAttnThreads;
    __shared__ v4i lds_mem[kAttnWaves * 16 * kLdsRow / 4];
    v4i* lds_q = lds_mem;                              // the queries' digits, then
    float* lds_o = reinterpret_cast<float*>(lds_mem);  // the waves' sums
    __shared__ float lds_ml[kAttnWaves][2][16];
    __shared__ int64_t lds_off[kAttnWaves][2][S::TK];
    __shared__ v4f lds_scale[kAttnWaves][2][S::TK / 4];  // of a tile's keys, of its values
    __shared__ int lds_last;
    __shared__ int64_t lds_ends[kAttnPlanRows];
    // Neighbouring shares of one head go to one XCD: units of a sequence then find
    // its positions in that XCD's L2
    const int id = xcd_remap(blockIdx.y * gridDim.x + blockIdx.x, gridDim.x * gridDim.y);
    const int heads = (unsigned)id / gridDim.x, share = id - heads * gridDim.x;
    const AttnLine<true, true> line(call.a, call.pl, lds_ends);
    if (share >= line.x) return;
    int64_t at = line.begin(share);
    const int64_t to_step = line.begin(share + 1);
    for (int r = line.row_at(at); at < to_step; ++r) {
        int64_t row_end;
        const AttnSeg it = line.segment(r, at, to_step, &row_end);
        at = row_end;
        // The arguments and the thread, opaque to the compiler: it would compute
        // everything that follows from them before the first segment, 1.4 us for
        // a call that has but one, and spill it
        typedef const __attribute__((address_space(4))) Attn8Call* Kernarg;
        Kernarg again = (Kernarg)__builtin_amdgcn_kernarg_segment_ptr();
        int tid = threadIdx.x;
        asm volatile("" : "+s"(again), "+v"(tid));
        const Attn8Call& k = *(const Attn8Call*)again;
        const AttnArgs& a = k.a;
        const AttnPlan& pl = k.pl;
        const KvView& c = a.c;
        const int D = c.D, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
        const int n = lane & 15, g = lane >> 4;
        const bool fast = D >= 16;
        const AttnUnit unit = attn_unit(a, r);
        const int hk = pl.tiles == 1 ? heads : fast_quot(heads, k.by_tiles);
        Attn8Cols cols;
        cols.row = unit.row;
        cols.G = k.G;
        cols.by_group = k.by_group;
        cols.several = a.unit_rows > 1;
        cols.h0 = hk * k.G + (heads - hk * pl.tiles) * 16;
        cols.n = cols.several ? unit.rows * k.G : min(16, hk * k.G + k.G - cols.h0);
        const int ntiles = it.p1 > it.p0 ? (it.p1 - it.p0 + S::TK - 1) / S::TK : 0;

        float m = -INFINITY, l = 0.0f;
        bool plain = !fast;
        v4f o[S::UE];
#pragma unroll
        for (int i = 0; i < S::UE; ++i) o[i] = v4f{0.0f, 0.0f, 0.0f, 0.0f};

        if (fast && ntiles > 0) {
            const int8_t* kc = static_cast<const int8_t*>(c.k);
            const int8_t* vc = static_cast<const int8_t*>(c.v);
            // byte offsets of the lane's pieces in a key's and a value's row
            int kd[S::KS];
#pragma unroll
            for (int s = 0; s < S::KS; ++s) kd[s] = min(16 * (4 * s + g), D - 16);
            const int vd = min(S::UE * n, D - S::UE);
            const AttnPlace own = cols(n < cols.n ? n : 0);
            // What the lane's column sees, and what every column of the unit does
            const int len = n < cols.n ? kv_length(c, a.lengths[own.row]) : it.n + it.gap;
            int least = len, most = len;
            if (cols.several) {
                for (int x = 1; x < 16; x <<= 1) {
                    least = min(least, __shfl_xor(least, x));
                    most = max(most, __shfl_xor(most, x));
                }
            }

            v4i kr[S::NT][S::KS];
            int vr[S::NJ][S::UE / 4];
            float ks_next = 0.0f, vs_next = 0.0f;  // scales of the lane's position
            uint64_t there = 0;                    // positions of the tile that exist
            const int8_t* vcol = vc + vd;
            const int8_t* kcol[S::KS];
#pragma unroll
            for (int s = 0; s < S::KS; ++s) kcol[s] = kc + kd[s];
            auto pos = [&](int i, int x) { return attn_pos<true>(a, it.gap, it.p0 + i * S::TK + x); };
            auto entry = [&](int i) {  // the lane's table entry of tile i
                const int x = min(it.p0 + i * S::TK + lane, it.p1 - 1);
                return c.table[(int64_t)it.seq * c.ldt + kv_page_of(c, attn_pos<true>(a, it.gap, x))];
            };
            // Row offsets of a tile's positions, one lane each, through the wave's
            // LDS (0: no position there), and the scales; whether every column
            // sees all of them
            auto offsets = [&](int i, int e) {
                const int p = pos(i, lane), slot = kv_slot(c, p);
                const bool in = ((unsigned)e < (unsigned)c.num_pages) & (it.p0 + i * S::TK + lane < it.p1);
                const int64_t pg = in ? e : 0, off = pg * c.sp + slot * c.ss + hk * c.sh;
                lds_off[wave][(i / kAttnWaves) & 1][lane] = in ? off : 0;
                const int64_t sc = (pg * c.hkv + hk) * c.page + slot;
                ks_next = a.ks[sc];
                vs_next = a.vs[sc];
                there = __ballot(in);
                return __ballot(in & (p < least) & ((p < a.sink) | (p >= most - a.window))) == ~(uint64_t)0;
            };
            auto load_k = [&](int i) {
                const int64_t* of = lds_off[wave][(i / kAttnWaves) & 1];
#pragma unroll
                for (int t = 0; t < S::NT; ++t) {
                    const int64_t off = of[16 * t + n];
#pragma unroll
                    for (int s = 0; s < S::KS; ++s) kr[t][s] = *reinterpret_cast<const v4ib*>(kcol[s] + off);
                }
            };
            auto load_v = [&](int i) {
                const int64_t* of = lds_off[wave][(i / kAttnWaves) & 1];
#pragma unroll
                for (int j = 0; j < S::NJ; ++j) {
                    const int8_t* row = vcol + of[16 * (j / 4) + 4 * g + j % 4];
                    if constexpr (S::UE == 16) {
                        const v4i x = __builtin_nontemporal_load(reinterpret_cast<const v4ib*>(row));
#pragma unroll
                        for (int u = 0; u < 4; ++u) vr[j][u] = x[u];
                    } else if constexpr (S::UE == 8) {
                        const v2i x = __builtin_nontemporal_load(reinterpret_cast<const v2ib*>(row));
                        vr[j][0] = x[0];
                        vr[j][1] = x[1];
                    } else {
                        vr[j][0] = __builtin_nontemporal_load(reinterpret_cast<const v1ib*>(row));
                    }
                }
            };

            // The queries' digits as the lanes' operands, to LDS, a wave each
            // piece: column n, elements from min(16 (4 s + g), D - 16);
            // where pieces overlap (D no multiple of 16, or past D) the earlier
            // one counts, the later one holds zeros.
            const float* q = a.q + own.row * a.ldq + (int64_t)own.head * D;
            auto q_load = [&](int s, float* x) {
                const int nom = 16 * (4 * s + g), d = min(nom, D - 16);
#pragma unroll
                for (int i = 0; i < 16; i += 4) {
                    const v4f f = *reinterpret_cast<const v4fu*>(q + d + i);
#pragma unroll
                    for (int e = 0; e < 4; ++e) x[i + e] = n < cols.n && d + i + e >= nom ? f[e] : 0.0f;
                }
            };
            // (table entries first, then the queries, then the first tile, which is
            // on its way while the queries become digits)
            int next_e = entry(wave);
            const int after_e = entry(wave + kAttnWaves);
            float x[S::KS][16], mx = 0.0f;
#pragma unroll
            for (int s = 0; s < S::KS; ++s) q_load(s, x[s]);
            // (unconditional, here and in the loop: a tile too many reads offset 0.
            // Behind loads under a condition the compiler waits for all of them)
            bool full = offsets(wave, next_e);
            next_e = after_e;
            load_k(wave);
            load_v(wave);
#pragma unroll
            for (int s = 0; s < S::KS; ++s)
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    plain |= !(fabsf(x[s][i]) < INFINITY);
                    mx = fmaxf(mx, fabsf(x[s][i]));
                    if (s && s == wave) x[0][i] = x[s][i];
                }
            mx = rows_max(mx);
            const int qk = mx < INFINITY ? digit_shift(mx) : 0;
            const float qs = ldexpf(k.scale2, -qk);
            if (wave < S::KS) {
                v4i dig[kDigits];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    unsigned b[4];
                    int w[kDigits];
#pragma unroll
                    for (int e = 0; e < 4; ++e) b[e] = digits_of((int)rintf(ldexpf(x[0][4 * i + e], qk)));
                    gather_digits(b, w);
#pragma unroll
                    for (int k = 0; k < kDigits; ++k) dig[k][i] = w[k];
                }
#pragma unroll
                for (int k = 0; k < kDigits; ++k) lds_q[(wave * kDigits + k) * 64 + lane] = dig[k];
            }
            __syncthreads();
            for (int i = wave; i < ntiles; i += kAttnWaves) {
                asm volatile("" ::: "memory");  // (the queries stay in LDS)
                const bool in = (there >> lane) & 1;
                const float ks1 = in ? ks_next : 0.0f, vs1 = in ? vs_next : 0.0f;
                reinterpret_cast<float*>(lds_scale[wave][0])[lane] = ks1;
                reinterpret_cast<float*>(lds_scale[wave][1])[lane] = vs1;
                plain |= !(fabsf(ks1) < INFINITY) | !((vs1 == 0.0f) | ((vs1 >= kLeastScale) & (vs1 < INFINITY)));
                // S of the tile
                float p[S::NJ];
#pragma unroll
                for (int t = 0; t < S::NT; ++t) {
                    v4i acc[kDigits];
#pragma unroll
                    for (int k = 0; k < kDigits; ++k) acc[k] = v4i{0, 0, 0, 0};
#pragma unroll
                    for (int s = 0; s < S::KS; ++s)
#pragma unroll
                        for (int k = 0; k < kDigits; ++k)
                            acc[k] = mfma(kr[t][s], lds_q[(s * kDigits + k) * 64 + lane], acc[k]);
                    const v4f ks = lds_scale[wave][0][4 * t + g];
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        p[4 * t + e] = fmaf((float)acc[2][e], 65536.0f, (float)((acc[1][e] << 8) + acc[0][e])) * (ks[e] * qs);
                    // (here, and not where they are needed: the sums would wait in
                    // three times the registers)
                    asm volatile("" : "+v"(p[4 * t]), "+v"(p[4 * t + 1]), "+v"(p[4 * t + 2]), "+v"(p[4 * t + 3]));
                }
                // the next tile's keys, in flight under this tile's softmax and values
                const bool was_full = full;
                const uint64_t was_there = there >> (4 * g);
                full = offsets(i + kAttnWaves, next_e);
                next_e = entry(i + 2 * kAttnWaves);
                load_k(i + kAttnWaves);
                if (!was_full) {
#pragma unroll
                    for (int j = 0; j < S::NJ; ++j) {
                        const int x = 16 * (j / 4) + j % 4;
                        const bool in = (was_there >> x) & 1;
                        p[j] = (in & attn_sees(a, len, pos(i, 4 * g + x))) ? p[j] : -INFINITY;
                    }
                }
                float mt = m;
#pragma unroll
                for (int j = 0; j < S::NJ; ++j) mt = fmaxf(mt, p[j]);
                mt = rows_max(mt);
                if (__any(mt > m)) {
                    const float f = pow2(m - (mt == -INFINITY ? 0.0f : mt));
                    m = mt;
                    l *= f;
#pragma unroll
                    for (int x = 0; x < S::UE; ++x) o[x] *= f;
                }
                const float base = m == -INFINITY ? 0.0f : m;
                float wm = 0.0f;
#pragma unroll
                for (int t = 0; t < S::NT; ++t) {
                    const v4f vs = lds_scale[wave][1][4 * t + g];
#pragma unroll
                    for (int j = 4 * t; j < 4 * t + 4; ++j) {
                        p[j] = pow2(p[j] - base);
                        l += p[j];
                        p[j] *= vs[j % 4];
                        wm = fmaxf(wm, p[j]);
                        asm volatile("" : "+v"(l));
                    }
                }
                // The weights' digits: p 2^k + 0x808080 is a whole number from
                // 2^23 up to 2^24, so the float's last bits are its digits, the
                // upper one as it is
                wm = rows_max(wm);
                const int pk = digit_shift(wm);
                const float up = ldexpf(1.0f, pk), down = ldexpf(1.0f, -pk);
                v4i pd[kDigits];
#pragma unroll
                for (int t = 0; t < S::NT; ++t) {
                    unsigned b[4];
                    int w[kDigits];
#pragma unroll
                    for (int e = 0; e < 4; ++e) b[e] = __float_as_uint(fmaf(p[4 * t + e], up, 8421504.0f));
                    gather_digits(b, w);
                    pd[0][t] = w[0] ^ (int)0x80808080;
                    pd[1][t] = w[1] ^ (int)0x80808080;
                    pd[2][t] = w[2];
                }
                const float down16 = down * 65536.0f;
#pragma unroll
                for (int u = 0; u < S::UE / 4; ++u) {
                    __builtin_amdgcn_sched_barrier(0);  // (or all columns are transposed first, and spilled)
                    int col[S::NT][4];
#pragma unroll
                    for (int t = 0; t < S::NT; ++t) {
                        const int x[4] = {vr[4 * t][u], vr[4 * t + 1][u], vr[4 * t + 2][u], vr[4 * t + 3][u]};
                        transpose4(x, col[t]);
                    }
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const v4i cv = {col[0][e], col[1][e], col[2][e], col[3][e]};
                        const v4i zero = {0, 0, 0, 0};
                        const v4i d2 = mfma(cv, pd[2], zero), d1 = mfma(cv, pd[1], zero), d0 = mfma(cv, pd[0], zero);
                        v4f& sum = o[4 * u + e];
#pragma unroll
                        for (int y = 0; y < 4; ++y)
                            sum[y] = fmaf((float)d2[y], down16, fmaf((float)((d1[y] << 8) + d0[y]), down, sum[y]));
                        asm volatile("" : "+v"(sum));
                    }
                }
                load_v(i + kAttnWaves);
            }
            l = rows_sum(l);
        }

        // The waves' sums, relative to the largest maximum: four elements of a
        // column a thread, kItems times
        v4f sum[kItems];
        auto at_item = [&](int j, int* h, int* d) {
            const int x = tid + kAttnThreads * j;
            *h = x / (DP / 4);
            *d = x % (DP / 4) * 4;
            return *h < cols.n && *d < D;
        };
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
            for (int y = 0; y < 4; ++y) {
                const int nom = S::UE * (4 * g + y);
                float* to = lds_o + (wave * 16 + n) * kLdsRow + nom;
                if (nom + S::UE <= D) {
#pragma unroll
                    for (int e = 0; e < S::UE; e += 4)
                        *reinterpret_cast<v4f*>(to + e) = v4f{o[e][y], o[e + 1][y], o[e + 2][y], o[e + 3][y]} * f;
                } else {  // a piece that begins at D - UE
#pragma unroll
                    for (int e = 0; e < S::UE; ++e)
                        if (D - S::UE + e >= nom) lds_o[(wave * 16 + n) * kLdsRow + D - S::UE + e] = o[e][y] * f;
                }
            }
            __syncthreads();
            if (tid < 16) {
                float lt = 0.0f;
                for (int w = 0; w < kAttnWaves; ++w)
                    lt += lds_ml[w][1][n] * pow2(lds_ml[w][0][n] - (mm == -INFINITY ? 0.0f : mm));
                lds_ml[0][0][n] = mm;
                lds_ml[0][1][n] = lt;
                plain |= n < cols.n && !(mm < INFINITY && lt < INFINITY);
            }
#pragma unroll
            for (int j = 0; j < kItems; ++j) {
                int h, d;
                if (!at_item(j, &h, &d)) continue;
                sum[j] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int w = 0; w < kAttnWaves; ++w)
                    sum[j] += *reinterpret_cast<const v4f*>(lds_o + (w * 16 + h) * kLdsRow + d);
#pragma unroll
                for (int e = 0; e < 4; ++e) plain |= d + e < D && !(fabsf(sum[j][e]) < INFINITY);
            }
        }
        // (A segment of nothing but holes has a maximum of -inf, sums of 0, and is
        // done.)
        if (__syncthreads_or(plain)) {
            attn8_plain(a, it, hk, cols, k.scale2, lds_o, &lds_ml[0][0][0], kLdsRow);
#pragma unroll
            for (int j = 0; j < kItems; ++j) {
                int h, d;
                if (at_item(j, &h, &d)) sum[j] = *reinterpret_cast<const v4f*>(lds_o + h * kLdsRow + d);
            }
        }

        if (it.nc == 1) {
#pragma unroll
            for (int j = 0; j < kItems; ++j) {
                int h, d;
                if (at_item(j, &h, &d)) attn8_out(a, cols(h), d, sum[j], lds_ml[0][1][h]);
            }
            if (a.lse && tid < cols.n) {
                const AttnPlace w = cols(n);
                a.lse[(int64_t)w.row * a.hq + w.head] = row_lse(lds_ml[0][0][n], lds_ml[0][1][n]);
            }
        } else {
            const int64_t slot = (int64_t)share + r, item = slot * pl.hy + heads;
#pragma unroll
            for (int j = 0; j < kItems; ++j) {
                int h, d;
                if (at_item(j, &h, &d)) attn8_part(pl, item, h, d, D, sum[j]);
            }
            if (tid < cols.n) st2_device(pl.part_ml + (item * 16 + n) * 2, lds_ml[0][0][n], lds_ml[0][1][n]);
            // its group's segments, then the groups: of 16, and of 32 where 16 of 16
            // would not do (16384 positions 20.6 us, in groups of 32 23.8; 131072
            // 58.5 and 60.2; 3000 16.8 and 16.1)
            const int size = it.nc <= 256 ? 16 : kJoinGroup, mine = (int)(slot - it.slot) & ~(size - 1);
            const int64_t g0 = it.slot + mine;
            const int groups = (it.nc + size - 1) / size;
            int64_t from = g0;
            int cnt = min(size, it.nc - mine), every = 1;
            unsigned* count = pl.count + g0 * pl.hy + heads;
#pragma unroll 1
            while (attention_count(count, cnt, &lds_last)) {
                const bool last = groups == 1 || every > 1;
                attn8_join<DP>(a, pl, cols, tid, heads, from, every, cnt, last, lds_o);
                if (last) break;
                from = it.slot;
                cnt = groups;
                every = size;
                count = pl.tops + (int64_t)r * pl.hy + heads;
            }
        }
        __syncthreads();
    }
}

namespace {

// Rows of one sequence that share a pass over the cache.
int unit_rows(const AttnArgs& a) {
    const int G = a.hq / a.c.hkv;
    return G > 16 ? 1 : std::min(a.tokens, 16 / G);
}
// Workgroups per compute unit, as the registers allow: three of D = 128 spill (131072
// positions 75 us, two 56), two of D = 64 are no slower for one row (38 us) and
// slower for 64 (69.5, three 65).
int resident(int D) { return D > 128 ? 1 : (D > 64 ? 2 : 3); }

AttnPlan make_plan(const AttnArgs& a, int cus) {
    AttnPlan pl = plan_attention(a, cus, unit_rows(a), resident(a.c.D));
    // (the line keeps 64 units in the lanes of a wave)
    pl.parts = pl.units <= 64 && 2 * pl.units <= pl.shares;
    return pl;
}

}  // namespace

size_t attention8_workspace(const AttnArgs& a, int cus, size_t* counters) {
    AttnPlan pl = make_plan(a, cus);
    *counters = attention_counters(a, pl);
    return place_attention(a, &pl, attention_splits(a, pl), nullptr);
}

hipError_t launch_paged_attention8(AttnArgs a, int cus, void* ws, void* counters, hipStream_t s) {
    a.unit_rows = unit_rows(a);
    a.units = (a.tokens + a.unit_rows - 1) / a.unit_rows;
    a.by_units = fast_div(a.units);
    AttnPlan pl = make_plan(a, cus);
    attention_memory(a, &pl, ws, counters);
    const dim3 grid((unsigned)pl.shares, (unsigned)pl.hy), block(kAttnThreads);
    const Attn8Call call = {a,
                            pl,
                            (float)((double)a.scale * 1.4426950408889634),
                            a.hq / a.c.hkv,
                            fast_div(a.hq / a.c.hkv),
                            fast_div(pl.tiles)};
    if (a.c.D <= 64)
        attention8_kernel<64><<<grid, block, 0, s>>>(call);
    else if (a.c.D <= 128)
        attention8_kernel<128><<<grid, block, 0, s>>>(call);
    else
        attention8_kernel<256><<<grid, block, 0, s>>>(call);
    return hipGetLastError();
}

}  // namespace xt
