// select.hip -- block means, and the blocks that every query selects.
//
//   mean[b] = sum of the block's keys / their number, summed in 64 bits and rounded once to the keys' type
//   score(t, b) = (sum over the group's heads of q[t, h]) . mean[b]
// A score decides which blocks a query sees, so two scores that differ only by rounding must still order the same way
// everywhere: they are compared in 64 bits.
#include "common.h"

namespace nsp {
namespace lm {

// ---- means -----------------------------------------------------------------------------------------------------------------
// One workgroup per (block, key head): eight neighbouring elements a lane, rows side by side, joined in LDS in a fixed order.
// Bound by reading K once: 16384 keys of 8 heads of 128, bf16, 10 us (3.4 TB/s); the newest block of 16 conversations 4 us.
template <class T>
__global__ void __launch_bounds__(256) k_block_means(const Geometry G, const T *__restrict__ k, T *__restrict__ means, int last, int per_seq)
{
    __shared__ double part[256 * 8];
    const int g = (int)(group_id() % G.kv_heads);
    const long long rest = group_id() / G.kv_heads;
    Seq sq;
    int b;
    if (per_seq > 0) {
        if (rest / per_seq >= G.n_seq) return;
        sq = seq_at(G, (int)(rest / per_seq));
        b = (int)(rest % per_seq);
        if (last > 0) b += (sq.k_len > last ? sq.k_len - last : 0) / G.block;
        if ((long long)b * G.block >= sq.k_len) return;
    } else if (!block_of_mean_row(G, rest, sq, b)) {
        return;
    }
    const int n = sq.k_len - b * G.block < G.block ? sq.k_len - b * G.block : G.block;
    const T *p;
    T *o;
    if (G.page_size > 0) {
        const long long page = page_of_block(G, sq.s, b);
        if (page < 0) return;
        p = k + page * G.k_page + (long long)(b % G.per_page) * G.block * G.k_row;
        o = means + (page * G.per_page + b % G.per_page) * G.kv_heads * G.head_dim;
    } else {
        p = k + (sq.k_base + (long long)b * G.block) * G.k_row;
        o = means + (mean_base(G, sq) + b) * G.kv_heads * G.head_dim;
    }
    p += (long long)g * G.k_head;
    o += (long long)g * G.head_dim;
    const int wide = G.head_dim / 8;        // lanes a row
    const int rows = 256 / wide;            // rows side by side
    const int r0 = (int)threadIdx.x / wide, d0 = ((int)threadIdx.x % wide) * 8;
    double acc[8] = {};
    if (r0 < rows) {
        for (int r = r0; r < n; r += rows) {
            typedef __attribute__((ext_vector_type(8))) T T8;
            const T8 x = __builtin_bit_cast(T8, frag_load(p + (long long)r * G.k_row + d0));
#pragma unroll
            for (int i = 0; i < 8; i++) acc[i] += (double)x[i];
        }
#pragma unroll
        for (int i = 0; i < 8; i++) part[r0 * G.head_dim + d0 + i] = acc[i];
    }
    __syncthreads();
    const int side = rows < n ? rows : n;
    for (int d = threadIdx.x; d < G.head_dim; d += 256) {
        double s = 0;
        for (int r = 0; r < side; r++) s += part[r * G.head_dim + d];
        o[d] = (T)(s / n);
    }
}

// ---- selection ---------------------------------------------------------------------------------------------------------------
// Scores are computed in 32 bits with a bound of their error,
//   |score32 - score| <= off = (D + group + 8) 2^-24 |sum_h |q_h|| max_b |mean_b|      (Cauchy-Schwarz over the products),
// and the need-th best 32-bit score a is found by bisection.  A block above a + 2 off is among the best whatever the errors
// are, one below a - 2 off is not; what lies between is scored again in 64 bits, wavefront by block, if not all of it is wanted.
// Rows whose bound is no finite number (NaN, infinities, overflow) or whose band is wide (many equal scores) take the plain way:
// every score in 64 bits and a search per selected block.
constexpr int kWidest = 256;

struct Competition {  // the blocks lo .. hi - 1 compete for `need` places
    int eligible, lo, hi, need;
};
__device__ inline Competition competition(const Geometry &G, const Seq &sq, int i, int first, int local)
{
    Competition c;
    if (G.causal) {
        const int pos = sq.k_len - sq.q_len + i;
        c.eligible = pos < 0 ? 0 : pos / G.block + 1;
    } else {
        c.eligible = (sq.k_len + G.block - 1) / G.block;
    }
    c.lo = first;
    c.hi = c.eligible > G.width ? c.eligible - local : 0;
    c.need = G.width - first - local;
    return c;
}
// first element of a block's mean for key head g; NULL where the page table names no page
template <class T> __device__ inline const T *mean_of_block(const Geometry &G, const Seq &sq, const T *means, int g, int b)
{
    long long m;
    if (G.page_size > 0) {
        const long long page = page_of_block(G, sq.s, b);
        if (page < 0) return nullptr;
        m = page * G.per_page + b % G.per_page;
    } else {
        m = mean_base(G, sq) + b;
    }
    return means + (m * G.kv_heads + g) * G.head_dim;
}

// The plain way, by a whole workgroup: `cap` scores at a time beside the best so far.
struct Plain {
    double best_score[kWidest], qsum[256];
    int wave_at[16], best_name[kWidest];
};
template <class T>
__device__ void select_plain(const Geometry &G, const Seq &sq, int t, int g, const Competition &c, const T *q, const T *means, int *row,
                             Plain &pl, char *space, int bytes)
{
    const int tid = threadIdx.x, threads = blockDim.x;
    const int slots = bytes / 12, cap = slots - kWidest;
    double *score = (double *)space;
    int *name = (int *)(space + 8 * (size_t)slots);
    __syncthreads();
    for (int d = tid; d < G.head_dim; d += threads) {
        double s = 0;
        for (int h = 0; h < G.group; h++) s += (double)to_f32(q[(long long)t * G.q_row + (long long)(g * G.group + h) * G.q_head + d]);
        pl.qsum[d] = s;
    }
    __syncthreads();
    int have = 0;
    for (int c0 = c.lo; c0 < c.hi && c.need > 0; c0 += cap) {
        const int n = c.hi - c0 < cap ? c.hi - c0 : cap;
        for (int x = tid; x < have; x += threads) {
            score[x] = pl.best_score[x];
            name[x] = pl.best_name[x];
        }
        for (int x = tid; x < n; x += threads) {
            const T *p = mean_of_block(G, sq, means, g, c0 + x);
            double s = -INFINITY;
            if (p) {
                s = 0;
                for (int d = 0; d < G.head_dim; d++) s += pl.qsum[d] * (double)to_f32(p[d]);
                if (s != s) s = -INFINITY;
            }
            score[have + x] = s;
            name[have + x] = c0 + x;
        }
        __syncthreads();
        const int total = have + n;
        const int take = c.need < total ? c.need : total;
        for (int r = 0; r < take; r++) {
            double bs = -INFINITY;
            int bn = 0x7fffffff, at = -1;
            for (int x = tid; x < total; x += threads)
                if (name[x] >= 0 && (score[x] > bs || (score[x] == bs && name[x] < bn))) {
                    bs = score[x];
                    bn = name[x];
                    at = x;
                }
            for (int d = 32; d > 0; d >>= 1) {
                const double os = __shfl_xor(bs, d);
                const int on = __shfl_xor(bn, d), oa = __shfl_xor(at, d);
                if (os > bs || (os == bs && on < bn)) {
                    bs = os;
                    bn = on;
                    at = oa;
                }
            }
            if ((tid & 63) == 0) pl.wave_at[tid >> 6] = at;
            __syncthreads();
            if (tid == 0) {
                int pick = -1;
                for (int w = 0; w < threads >> 6; w++) {
                    const int a = pl.wave_at[w];
                    if (a < 0) continue;
                    if (pick < 0 || score[a] > score[pick] || (score[a] == score[pick] && name[a] < name[pick])) pick = a;
                }
                pl.best_score[r] = score[pick];
                pl.best_name[r] = name[pick];
                name[pick] = -1;
            }
            __syncthreads();
        }
        have = take;
    }
    for (int x = tid; x < have; x += threads) {
        int r = 0;
        for (int y = 0; y < have; y++) r += pl.best_name[y] < pl.best_name[x];
        row[c.lo + r] = pl.best_name[x];
    }
    __syncthreads();
}

// The places that no score decides.  Returns whether a competition is left.
__device__ inline bool write_forced(const Geometry &G, const Competition &c, int first, int local, int *row, int lane, int lanes)
{
    if (c.eligible <= G.width) {
        for (int x = lane; x < G.width; x += lanes) row[x] = x < c.eligible ? x : -1;
        return false;
    }
    for (int x = lane; x < first; x += lanes) row[x] = x;
    for (int x = lane; x < local; x += lanes) row[G.width - local + x] = c.hi + x;
    return c.need > 0;
}

__device__ inline unsigned order_key(float x)
{
    const unsigned u = __float_as_uint(x);
    return (u >> 31) ? ~u : u | 0x80000000u;
}
__device__ inline float key_value(unsigned k) { return __uint_as_float((k >> 31) ? k & 0x7fffffffu : ~k); }

// One wavefront: the best c.need of score[c.lo .. c.hi) (LDS, finite), each off by at most `off`; false: take the plain way.
// NV > 0: at most 64 NV scores, which stay in registers.
template <class T, int NV>
__device__ bool select_wave(const Geometry &G, const Seq &sq, int t, int g, const Competition &c, const T *q, const T *means, float off,
                            float *score, int *row)
{
    const int lane = lane_id();
    // 2 off, rounded up through the additions below
    const float band = 2.0f * off;
    if (!(band < 1e30f)) return false;
    const int n = c.hi - c.lo;
    float kept[NV > 0 ? NV : 1];
    if constexpr (NV > 0) {
#pragma unroll
        for (int v = 0; v < NV; v++) kept[v] = 64 * v + lane < n ? score[c.lo + 64 * v + lane] : -INFINITY;
    }
    // f(score, its place) for 64 scores at a time; the places behind the last hold -inf
    auto each = [&](auto f) {
        if constexpr (NV > 0) {
#pragma unroll
            for (int v = 0; v < NV; v++)
                if (64 * v < n) f(kept[v], 64 * v + lane);
        } else {
            for (int x = lane; x - lane < n; x += 64) f(x < n ? score[c.lo + x] : -INFINITY, x);
        }
    };
    float lo = INFINITY, hi = -INFINITY;
    each([&](float s, int x) {
        lo = fminf(lo, x < n ? s : INFINITY);
        hi = fmaxf(hi, s);
    });
    lo = -wave_max(-lo);
    hi = wave_max(hi);
    // count(>= key_lo) >= need, count(>= key_hi) < need; by value while that halves well, then by the numbers' bits
    unsigned key_lo = (unsigned)uniform((int)order_key(lo)), key_hi = (unsigned)uniform((int)order_key(hi)) + 1;
    int m_lo = n;
    for (int step = 0; key_hi - key_lo > 1 && m_lo != c.need; step++) {
        unsigned key = key_lo + (key_hi - key_lo) / 2;
        if (step < 14) {
            const float mid = 0.5f * key_value(key_lo) + 0.5f * key_value(key_hi - 1);
            const unsigned k = (unsigned)uniform((int)order_key(mid));
            if (k > key_lo && k < key_hi) key = k;
        }
        const float mid = key_value(key);
        int m = 0;
        each([&](float s, int) { m += __popcll(__ballot(s >= mid)); });
        if (m >= c.need) {
            key_lo = key;
            m_lo = m;
        } else {
            key_hi = key;
        }
    }
    // a: the need-th best
    const float at_least = key_value(key_lo);
    float a = INFINITY;
    each([&](float s, int) { a = s >= at_least ? fminf(a, s) : a; });
    a = -wave_max(-a);
    const float slack = band + 4.0f * 5.9604645e-8f * (fabsf(a) + band);
    const float above = a + slack, below = a - slack;
    int sure = 0, between = 0;
    each([&](float s, int) {
        sure += __popcll(__ballot(s > above));
        between += __popcll(__ballot(s >= below && s <= above));
    });
    const int places = c.need - sure;
    if (between != places) {
        if (between > 64) return false;
        double mine[4];  // the group's summed queries at columns lane, lane + 64, ...
        for (int z = 0; z < 4; z++) {
            const int d = lane + 64 * z;
            mine[z] = 0;
            if (d < G.head_dim)
                for (int h = 0; h < G.group; h++) mine[z] += (double)to_f32(q[(long long)t * G.q_row + (long long)(g * G.group + h) * G.q_head + d]);
        }
        double es = 0;
        int eb = -1, k = 0;
        for (int x0 = c.lo; x0 < c.hi; x0 += 64) {
            const float s = x0 + lane < c.hi ? score[x0 + lane] : -INFINITY;
            unsigned long long m = __ballot(s >= below && s <= above);
            while (m) {
                const int b = x0 + __builtin_ctzll(m);
                m &= m - 1;
                const T *p = mean_of_block(G, sq, means, g, b);
                double e = 0;
                for (int z = 0; z < 4; z++) {
                    const int d = lane + 64 * z;
                    if (d < G.head_dim && p) e += mine[z] * (double)to_f32(p[d]);
                }
#pragma unroll
                for (int d = 1; d < 64; d <<= 1) e += __shfl_xor(e, d);
                if (lane == k) {
                    es = e;
                    eb = b;
                }
                k++;
            }
        }
        int better = 0;
        for (int y = 0; y < k; y++) {
            const double os = __shfl(es, y);
            const int ob = __shfl(eb, y);
            better += os > es || (os == es && ob < eb);
        }
        if (eb >= 0) score[eb] = better < places ? INFINITY : -INFINITY;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        if constexpr (NV > 0) {
#pragma unroll
            for (int v = 0; v < NV; v++) kept[v] = 64 * v + lane < n ? score[c.lo + 64 * v + lane] : -INFINITY;
        }
    }
    int at = c.lo;
    each([&](float s, int x) {
        const bool in = s >= below;
        const unsigned long long m = __ballot(in);
        if (in) row[at + __popcll(m & ((1ULL << lane) - 1))] = c.lo + x;
        at += __popcll(m);
    });
    return true;
}

// The bound of a row's scores from the norms; not finite where the scores may not be.  The squares' 1e-30 stands for what underflows:
// numbers whose square is lost, and products below the smallest normal number (at most head_dim 2^-126 in all).
__device__ inline float score_off(const Geometry &G, float q_norm2, float mean_norm2)
{
    return (G.head_dim + G.group + 8) * 5.9604645e-8f * 1.01f * sqrtf(q_norm2 + 1e-30f) * sqrtf(mean_norm2 + 1e-30f);
}
__device__ inline float max_or_nan(float a, float b) { return (b > a || b != b) ? b : a; }

// Prompts: one workgroup per (16 query rows, key head).  The rows' summed queries are the right operand, sixteen block means the left,
// as 32-bit matrix products; the four wavefronts take every fourth tile of blocks, then four rows each for the
// choice.  The scores stay in LDS (CAP blocks a row: LDS leaves four workgroups a CU for 256, two for 768, one for 2048).
// 16384 queries of 32 heads of 128, 256 blocks, bf16: 228 us, half of it the search for the border (its compares and counts), 13 us the products.
template <class T, int KS, int CAP>
__global__ void __launch_bounds__(256)
    k_select_rows(const Geometry G, int first, int local, const T *__restrict__ q, const T *__restrict__ means, int *__restrict__ idx)
{
    constexpr int LQ = 32 * KS + 4, LS = CAP + 4;
    __shared__ float qs[16 * LQ];
    __shared__ __align__(16) float score[16 * LS];
    __shared__ float q_norm2[16], mean_norm2[16];  // of the wavefront
    __shared__ int plain_row[16];
    __shared__ Plain pl;
    const int lane = lane_id(), col = lane & 15, quad = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const int all = (G.q_rows + 15) / 16 * G.kv_heads, mine = all - 1 - (int)group_id();
    if (mine < 0) return;
    const int g = mine % G.kv_heads;
    // the last rows, which see most, begin first
    const int t0 = mine / G.kv_heads * 16;
    const int t1 = t0 + 16 < G.q_rows ? t0 + 16 : G.q_rows;
    if (threadIdx.x < 16) plain_row[threadIdx.x] = 0;
    // the group's summed queries, and the norm of the sum of their absolute values
    {
        const int r = (int)threadIdx.x >> 4, l16 = (int)threadIdx.x & 15;
        float n2 = 0.f;
        for (int d0 = l16 * 8; d0 < 32 * KS; d0 += 128) {
            float s[8] = {}, n[8] = {};
            if (t0 + r < t1 && d0 < G.head_dim)
                for (int h = 0; h < G.group; h++) {
                    typedef __attribute__((ext_vector_type(8))) T T8;
                    const T8 x = __builtin_bit_cast(T8, frag_load(q + (long long)(t0 + r) * G.q_row + (long long)(g * G.group + h) * G.q_head + d0));
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        s[i] += (float)x[i];
                        n[i] += fabsf((float)x[i]);
                    }
                }
#pragma unroll
            for (int i = 0; i < 8; i++) {
                qs[r * LQ + d0 + i] = s[i];
                n2 += n[i] * n[i];
            }
        }
#pragma unroll
        for (int d = 1; d < 16; d <<= 1) n2 += __shfl_xor(n2, d);
        if (l16 == 0) q_norm2[r] = n2;
    }
    __syncthreads();
    Frag<float> qf[KS];
#pragma unroll
    for (int z = 0; z < KS; z++) {
        const float *p = qs + col * LQ + 32 * z + 8 * quad;
        qf[z] = frag_load(p);
    }
    // the rows may belong to several sequences: one after the other
    for (int a = t0; a < t1;) {
        Seq sq;
        const int i0 = seq_of_query(G, a, sq);
        if (i0 < 0) {
            a++;
            continue;
        }
        const int z = sq.q_base + sq.q_len < t1 ? (int)(sq.q_base + sq.q_len) : t1;
        const int hi = competition(G, sq, (int)(z - 1 - sq.q_base), first, local).hi;  // the last row's is the greatest
        float n2max = 0.f;
        for (int b0 = first / 16 * 16 + 16 * wave; b0 < hi; b0 += 64) {
            const int b = b0 + col;
            const T *p = b < hi ? mean_of_block(G, sq, means, g, b) : nullptr;
            const bool hidden = b < hi && !p;
            f32x4 s = f32x4{0, 0, 0, 0};
            float n2 = 0.f;
#pragma unroll
            for (int x = 0; x < KS; x++) {
                const int d = 32 * x + 8 * quad;
                typedef __attribute__((ext_vector_type(8))) T T8;
                T8 v{};
                if (p && d < G.head_dim) v = __builtin_bit_cast(T8, frag_load(p + d));
                Frag<float> f;
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    f.lo[i] = (float)v[i];
                    f.hi[i] = (float)v[4 + i];
                }
#pragma unroll
                for (int i = 0; i < 4; i++) n2 += f.lo[i] * f.lo[i] + f.hi[i] * f.hi[i];
                s = mma(f, qf[x], s);
            }
            // a block whose page is none scores lowest: the plain way sees to that
            n2max = max_or_nan(n2max, hidden ? NAN : quads_sum(n2));
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (b0 + 4 * quad + i < hi && t0 + col >= a && t0 + col < z) score[col * LS + b0 + 4 * quad + i] = s[i];
        }
#pragma unroll
        for (int d = 1; d < 16; d <<= 1) n2max = max_or_nan(n2max, __shfl_xor(n2max, d));
        if (lane == 0) mean_norm2[wave] = n2max;
        __syncthreads();
        const float m2 = max_or_nan(max_or_nan(mean_norm2[0], mean_norm2[1]), max_or_nan(mean_norm2[2], mean_norm2[3]));
        for (int t = a + ((wave - (a - t0)) & 3); t < z; t += 4) {
            const Competition c = competition(G, sq, (int)(t - sq.q_base), first, local);
            int *row = idx + ((long long)t * G.kv_heads + g) * G.width;
            if (!write_forced(G, c, first, local, row, lane, 64)) continue;
            if (!select_wave<T, CAP <= 768 ? CAP / 64 : 0>(G, sq, t, g, c, q, means, score_off(G, q_norm2[t - t0], m2), score + (t - t0) * LS, row))
                plain_row[t - t0] = 1;
        }
        __syncthreads();
        for (int t = a; t < z; t++)
            if (plain_row[t - t0])
                select_plain(G, sq, t, g, competition(G, sq, (int)(t - sq.q_base), first, local), q, means,
                             idx + ((long long)t * G.kv_heads + g) * G.width, pl, (char *)score, (int)sizeof(score));
        __syncthreads();
        a = z;
    }
}

// Single tokens: one workgroup per (query row, key head); sixteen lanes share a block's mean.  Bound by the way to memory, three times in a row
// (page, mean, choice): 16 conversations of up to 512 blocks 15 us.
constexpr int kOneCap = 32768;
template <class T>
__global__ void __launch_bounds__(1024)
    k_select_one(const Geometry G, int first, int local, const T *__restrict__ q, const T *__restrict__ means, int *__restrict__ idx)
{
    extern __shared__ __align__(16) float score[];
    __shared__ float norms[16];
    __shared__ int plain;
    __shared__ Plain pl;
    const int lane = lane_id(), l16 = lane & 15;
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const int g = (int)(group_id() % G.kv_heads), t = (int)(group_id() / G.kv_heads);
    if (t >= G.q_rows) return;
    Seq sq;
    const int i = seq_of_query(G, t, sq);
    if (i < 0) return;
    const Competition c = competition(G, sq, i, first, local);
    int *row = idx + ((long long)t * G.kv_heads + g) * G.width;
    if (!write_forced(G, c, first, local, row, (int)threadIdx.x, 1024)) return;
    typedef __attribute__((ext_vector_type(8))) T T8;
    float s[16] = {}, q2 = 0.f;
#pragma unroll
    for (int z = 0; z < 2; z++) {
        const int d = 128 * z + 8 * l16;
        float n[8] = {};
        if (d < G.head_dim)
            for (int h = 0; h < G.group; h++) {
                const T8 x = __builtin_bit_cast(T8, frag_load(q + (long long)t * G.q_row + (long long)(g * G.group + h) * G.q_head + d));
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    s[8 * z + e] += (float)x[e];
                    n[e] += fabsf((float)x[e]);
                }
            }
#pragma unroll
        for (int e = 0; e < 8; e++) q2 += n[e] * n[e];
    }
#pragma unroll
    for (int d = 1; d < 16; d <<= 1) q2 += __shfl_xor(q2, d);
    float n2max = 0.f;
    // four blocks at a time: their pages are all asked for, then their means, before any is used
    for (int b0 = c.lo + (int)(threadIdx.x >> 4); b0 < c.hi; b0 += 256) {
        const T *p[4];
        T8 x[4][2];
#pragma unroll
        for (int u = 0; u < 4; u++) {
            const int b = b0 + 64 * u;
            p[u] = b < c.hi ? mean_of_block(G, sq, means, g, b) : nullptr;
        }
#pragma unroll
        for (int u = 0; u < 4; u++)
#pragma unroll
            for (int z = 0; z < 2; z++) {
                const int d = 128 * z + 8 * l16;
                x[u][z] = T8{};
                if (p[u] && d < G.head_dim) x[u][z] = __builtin_bit_cast(T8, frag_load(p[u] + d));
            }
#pragma unroll
        for (int u = 0; u < 4; u++) {
            const int b = b0 + 64 * u;
            float dot = 0.f, n2 = 0.f;
#pragma unroll
            for (int z = 0; z < 2; z++)
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    dot += s[8 * z + e] * (float)x[u][z][e];
                    n2 += (float)x[u][z][e] * (float)x[u][z][e];
                }
#pragma unroll
            for (int d = 1; d < 16; d <<= 1) {
                dot += __shfl_xor(dot, d);
                n2 += __shfl_xor(n2, d);
            }
            if (b < c.hi) {
                n2max = max_or_nan(n2max, p[u] ? n2 : NAN);
                if (l16 == 0) score[b] = dot;
            }
        }
    }
#pragma unroll
    for (int d = 16; d < 64; d <<= 1) n2max = max_or_nan(n2max, __shfl_xor(n2max, d));
    if (lane == 0) norms[wave] = n2max;
    __syncthreads();
    if (wave == 0) {
        float m2 = norms[0];
        for (int w = 1; w < 16; w++) m2 = max_or_nan(m2, norms[w]);
        const float off = score_off(G, q2, m2);
        const bool done = c.hi - c.lo <= 512 ? select_wave<T, 8>(G, sq, t, g, c, q, means, off, score, row)
                                             : select_wave<T, 0>(G, sq, t, g, c, q, means, off, score, row);
        if (lane == 0) plain = !done;
    }
    __syncthreads();
    if (plain) select_plain(G, sq, t, g, c, q, means, row, pl, (char *)score, 8192 * 4);
}

// Sequences of more blocks than LDS holds scores for: the plain way for every row.
template <class T>
__global__ void __launch_bounds__(256)
    k_select_long(const Geometry G, int first, int local, const T *__restrict__ q, const T *__restrict__ means, int *__restrict__ idx)
{
    __shared__ __align__(16) char space[12 * 4096];
    __shared__ Plain pl;
    const int g = (int)(group_id() % G.kv_heads), t = (int)(group_id() / G.kv_heads);
    if (t >= G.q_rows) return;
    Seq sq;
    const int i = seq_of_query(G, t, sq);
    if (i < 0) return;
    const Competition c = competition(G, sq, i, first, local);
    int *row = idx + ((long long)t * G.kv_heads + g) * G.width;
    if (write_forced(G, c, first, local, row, (int)threadIdx.x, 256)) select_plain(G, sq, t, g, c, q, means, row, pl, space, (int)sizeof(space));
}

template <class T, int KS>
static void launch_rows(const Geometry &G, long long blocks, int first, int local, const void *q, const void *means, int *idx, hipStream_t st)
{
    const dim3 grid = groups(ceil_div(G.q_rows, 16) * G.kv_heads);
    if (blocks <= 256)
        launch((k_select_rows<T, KS, 256>), grid, dim3(256), 0, st, G, first, local, (const T *)q, (const T *)means, idx);
    else if (blocks <= 768)
        launch((k_select_rows<T, KS, 768>), grid, dim3(256), 0, st, G, first, local, (const T *)q, (const T *)means, idx);
    else
        launch((k_select_rows<T, KS, 2048>), grid, dim3(256), 0, st, G, first, local, (const T *)q, (const T *)means, idx);
}

template <class T>
static void launch_select(const Geometry &G, int first, int local, const void *q, const void *means, int *idx, hipStream_t st)
{
    // the most blocks a sequence can have, as far as the host knows
    const long long blocks = G.page_size > 0 ? G.table_stride * G.per_page : G.cu_k ? ceil_div(G.k_rows, G.block) : G.blocks_each;
    // sixteen rows together where there are enough to fill the machine and sequences have several (256 blocks, 8 key heads: 16 conversations of
    // 4 tokens 50 against 24 us row by row, 64 of 4 60 against 79, 16 of 16 over 1024 blocks 116 against 233, 4096 tokens 809 against 3405)
    if (blocks <= 2048 && G.q_rows / G.n_seq >= 4 && (long long)G.q_rows * G.kv_heads >= 1024) {
        if (G.head_dim <= 64) launch_rows<T, 2>(G, blocks, first, local, q, means, idx, st);
        else if (G.head_dim <= 128) launch_rows<T, 4>(G, blocks, first, local, q, means, idx, st);
        else launch_rows<T, 8>(G, blocks, first, local, q, means, idx, st);
        return;
    }
    const dim3 grid = groups((long long)G.q_rows * G.kv_heads);
    if (blocks <= kOneCap) {
        // the plain way wants 32 KB
        const size_t lds = blocks <= 8192 ? 8192 * 4 : (size_t)blocks * 4;
        if (lds > 65536) note_launch(hipFuncSetAttribute((const void *)k_select_one<T>, hipFuncAttributeMaxDynamicSharedMemorySize, kOneCap * 4));
        launch(k_select_one<T>, grid, dim3(1024), lds, st, G, first, local, (const T *)q, (const T *)means, idx);
    } else {
        launch(k_select_long<T>, grid, dim3(256), 0, st, G, first, local, (const T *)q, (const T *)means, idx);
    }
}

}  // namespace lm
}  // namespace nsp

extern "C" {

int nsparse_lm_block_means(const nsparse_lm_attn *a, const void *k, void *means, int last, void *stream)
{
    using namespace nsp::lm;
    clear_error();
    Geometry G;
    if (int rc = geometry(a, false, false, &G)) return rc;
    if (last < 0) return fail(NSPARSE_LM_EARG, "block_means: last must not be negative");
    if (G.k_rows == 0) return 0;
    if (!k || !means) return fail(NSPARSE_LM_EARG, "block_means: a required pointer is NULL");
    const int per16 = 16 / elem_size(a->dtype);
    for (int i = a->page_size > 0 ? 0 : 1; i < 3; i++)
        if (a->k_stride[i] % per16 || a->k_stride[i] < 0) return fail(NSPARSE_LM_EALIGN, "k strides must be multiples of 16 bytes");
    if (((uintptr_t)k | (uintptr_t)means) & 15) return fail(NSPARSE_LM_EALIGN, "block_means: k and means begin at multiples of 16 bytes");
    long long per_seq = 0, rows;
    // the most blocks a sequence can have
    const long long most = G.page_size > 0 ? G.table_stride * G.per_page : G.cu_k ? ceil_div(G.k_rows, G.block) : G.blocks_each;
    if (most == 0) return 0;  // tables without an entry
    if (last > 0) per_seq = (last - 1) / G.block + 2;
    if (per_seq > most || (G.page_size > 0 && per_seq == 0)) per_seq = most;
    rows = per_seq > 0 ? per_seq * G.n_seq : nsparse_lm_mean_rows(a);
    if (rows * G.kv_heads > kMostGroups) return fail(NSPARSE_LM_EARG, "block_means: blocks x heads out of range");
    if (rows == 0) return 0;
    const dim3 grid = groups(rows * G.kv_heads);
    hipStream_t st = (hipStream_t)stream;
    if (a->dtype == NSPARSE_LM_BF16)
        launch(k_block_means<__bf16>, grid, dim3(256), 0, st, G, (const __bf16 *)k, (__bf16 *)means, last, (int)per_seq);
    else if (a->dtype == NSPARSE_LM_F16)
        launch(k_block_means<_Float16>, grid, dim3(256), 0, st, G, (const _Float16 *)k, (_Float16 *)means, last, (int)per_seq);
    else
        launch(k_block_means<float>, grid, dim3(256), 0, st, G, (const float *)k, (float *)means, last, (int)per_seq);
    return launched("block_means");
}

int nsparse_lm_select_blocks(const nsparse_lm_attn *a, const void *q, const void *means, int *idx, void *stream)
{
    using namespace nsp::lm;
    clear_error();
    Geometry G;
    if (int rc = geometry(a, true, false, &G)) return rc;
    if (a->first < 0 || a->local < 0 || a->first > a->width || a->local > a->width || a->first + a->local > a->width)
        return fail(NSPARSE_LM_EARG, "select_blocks: first + local must not exceed width");
    if (G.causal && a->local < 1) return fail(NSPARSE_LM_EARG, "select_blocks: local must be at least 1 with causal");
    if (!G.causal && a->local != 0) return fail(NSPARSE_LM_EARG, "select_blocks: local must be 0 without causal");
    if (G.q_rows == 0) return 0;
    if (!q || !idx || (G.k_rows > 0 && !means)) return fail(NSPARSE_LM_EARG, "select_blocks: a required pointer is NULL");
    if (((uintptr_t)q | (uintptr_t)means) & 15) return fail(NSPARSE_LM_EALIGN, "select_blocks: q and means begin at multiples of 16 bytes");
    hipStream_t st = (hipStream_t)stream;
    if (a->dtype == NSPARSE_LM_BF16) launch_select<__bf16>(G, a->first, a->local, q, means, idx, st);
    else if (a->dtype == NSPARSE_LM_F16) launch_select<_Float16>(G, a->first, a->local, q, means, idx, st);
    else launch_select<float>(G, a->first, a->local, q, means, idx, st);
    return launched("select_blocks");
}
}
