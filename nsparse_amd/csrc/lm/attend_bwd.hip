// attend_bwd.hip -- gradient of attention over the listed blocks of keys.
//
//   p = exp(s - lse), delta = dout . out - dlse, ds = p (dout . v - delta)      (dlse: what comes back through the log-sum-exp)
//   dq = scale sum_j ds_j k_j          over the keys that the query's row lists: the pattern, one wavefront a row
//   dk = scale sum_t ds_t q_t, dv = sum_t p_t dout_t    over the queries that list the key's block: the transposed pattern
//
// The transposed pattern is a bitmap: for every key head and block one bit a query row, built by 64 rows a workgroup in
// LDS and written as whole words, so it needs no counting, no sort and no atomics on memory, and the order of
// the sums in dk and dv is the order of the rows, whatever the timing.  p and scale * ds are rounded to the inputs' type for the second
// products, whose operands in 32 bits would run at a seventh of the rate (with the scale, so that half precision overflows no sooner than the
// gradients themselves do).
#include "attend.h"

namespace nsp {
namespace lm {

// ---- dq (and delta) ----------------------------------------------------------------------------------------------------
// As the forward for prompts (attend_fwd.hip): the workgroup's rows are the columns of its products, the union of their blocks goes
// through LDS.  S^T = K Q^T and dP^T = V dO^T read K and V by rows, dQ^T = K^T dS^T reads K transposed.
// delta comes from the output as the forward rounded it.  That rounding matters where few keys share the weight, so workgroups with
// at most kExact keys in their union walk twice and take sum p (dout . v) from the first walk.  In single precision the
// probabilities are divided by their sum, which takes the rounding of the log-sum-exp out of them.
// A query with a single key (the first of a sequence) has p = 1 and ds = 0 whatever dout is; dout . v and delta differ by their roundings there, so
// such rows are counted out: dq = 0, and RowInfo tells dk.
// 32 keys a step and one set of columns a wavefront leave three wavefronts a SIMD, which hide each other's reads of LDS and the wait for
// the next tiles that stands before them (attend_fwd.hip), its bounds.  4096 rows of 32 heads of 128, 16 blocks each, bf16, against two sets and 64 keys a step (as the forward has where blocks allow):
// blocks of 64: 277 against 313 us, of 32: 195 against 318, of 16: 148 against 210.
constexpr int kExact = 256;
struct RowInfo {  // of a query row and head, for dk and dv
    float lse2, delta, inv;
    float single;  // 1: the row has one key, and its ds is 0
};
template <class T, int DP, bool WIDE>
__global__ void __launch_bounds__(256, DP * sizeof(T) <= 256 ? 2 : 1)
    k_attend_dq(const Geometry G, const T *__restrict__ q, const T *__restrict__ k, const T *__restrict__ v, const int *__restrict__ idx,
                const T *__restrict__ out, const float *__restrict__ lse, const T *__restrict__ dout, const float *__restrict__ dlse,
                T *__restrict__ dq, RowInfo *__restrict__ info, int slices, int per_tile)
{
    constexpr int KS = DP / 32, E = DP / 16, NG = 2 /* groups of sixteen keys a step */, kTile = NG * 16 * Tile<T, DP>::kPieces;
    __shared__ u32x4 kt[2][kTile], vt[2][kTile];
    __shared__ Union un;
    const int wave = uniform((int)(threadIdx.x >> 6));
    const int g = (int)(group_id() % G.kv_heads);
    const int rest = (int)(group_id() / G.kv_heads);
    const int slice = rest % slices;
    const int t0 = (rest / slices) * 4 * per_tile;
    const int t1 = t0 + 4 * per_tile < G.q_rows ? t0 + 4 * per_tile : G.q_rows;
    const int D = G.head_dim;
    const float sl2 = G.scale * kLog2e;

    for (int a = t0; a < t1;) {
        Seq sq;
        const int i0 = seq_of_query(G, a, sq);
        if (i0 < 0) {
            a++;
            continue;
        }
        const int z = sq.q_end < t1 ? sq.q_end : t1;
        const Column c0(G, g, slice, per_tile);
        const int col = c0.col, quad = c0.quad;
        // lane i's row for the walk; a column's row is number wave * per_tile + Column::sub
        const int t_mine = t0 + opaque(lane_id());
        const int limit = t_mine >= a && t_mine < z ? visible_keys(G, sq, (int)(t_mine - sq.q_base)) : 0;
        Frag<T> qf[KS], gf[KS];
        const int num = wave * per_tile + c0.sub;
        const bool on = c0.live && t0 + num >= a && t0 + num < z;
        int lim = pull(limit, num);
        if (!on) lim = 0;
        const int t = on ? t0 + num : a;
        const long long th = (long long)t * G.heads + c0.head;
        row_frags<T, KS, false>(gf, dout + th * D, quad, D, on);
        row_frags<T, KS, false>(qf, out + th * D, quad, D, on);
        float rounded = 0.f;
#pragma unroll
        for (int w = 0; w < KS; w++) rounded += frag_dot(gf[w], qf[w]);
        rounded = quads_sum(rounded);
        const float lse2 = on ? lse[th] * kLog2e : INFINITY;
        const auto through_lse = [&] { return dlse && on && lse2 != -INFINITY ? dlse[th] : 0.f; };
        rounded -= through_lse();
        row_frags<T, KS, false>(qf, q + (long long)t * G.q_row + (long long)c0.head * G.q_head, quad, D, on);
        const int count = z - a;
        const unsigned long long every = (count < 64 ? (1ULL << count) - 1 : ~0ULL) << (a - t0);
        unsigned long long todo = every, now = every;
        while (todo) {
            f32x4 o[E];
            float total = 0.f, with_dp = 0.f, delta = rounded;
            int keys = 0;  // that the column's row sees; 2 stands for more
#pragma unroll
            for (int j = 0; j < E; j++) o[j] = f32x4{0, 0, 0, 0};
            const int blocks = (read_lane(limit, 63 - __builtin_clzll(now)) + G.block - 1) / G.block;
            for (int b0 = 0; b0 < blocks; b0 += kRange) {
                union_build(un, G, idx, g, t0, now, limit, b0, blocks - b0 < kRange ? blocks - b0 : kRange, wave);
                const int steps = walk_steps<NG, WIDE>(G, un);
                if (steps == 0) continue;
                const bool exact = sizeof(T) == 2 && blocks <= kRange && steps * NG * 16 <= kExact;
                for (int pass = exact ? 0 : 1; pass < 2; pass++) {
                    Step<NG, WIDE> st;
                    walk_step<NG, WIDE>(st, G, sq, g, un, b0, limit, 0);
                    tile_load<T, DP, NG, WIDE>(kt[0], k, st.k_off, st, G.k_row, D);
                    tile_load<T, DP, NG, WIDE>(vt[0], v, st.v_off, st, G.v_row, D);
                    __syncthreads();
                    for (int step = 0; step < steps; step++) {
                        const int buf = step & 1;
                        Step<NG, WIDE> next = st;
                        if (step + 1 < steps) {
                            walk_step<NG, WIDE>(next, G, sq, g, un, b0, limit, step + 1);
                            tile_load<T, DP, NG, WIDE>(kt[buf ^ 1], k, next.k_off, next, G.k_row, D);
                            tile_load<T, DP, NG, WIDE>(vt[buf ^ 1], v, next.v_off, next, G.v_row, D);
                        }
                        const bool use = (st.any >> (wave * per_tile)) & ((1ULL << per_tile) - 1);
                        if (use) {
                            f32x4 s[2], d[2];
                            s[0] = s[1] = d[0] = d[1] = f32x4{0, 0, 0, 0};
                            pipelined<Frag<T>, 4 * KS, 4, 2>(
                                [&](int i) { return tile_frag<T, DP>(i < 2 * KS ? kt[buf] : vt[buf], 16 * (i / KS & 1) + col, i % KS, quad); },
                                [&](int i, const Frag<T> &f) {
                                    const int y = i / KS & 1;
                                    if (i < 2 * KS) s[y] = mma(f, qf[i % KS], s[y]);
                                    else d[y] = mma(f, gf[i % KS], d[y]);
                                });
#pragma unroll
                            for (int y = 0; y < 2; y++) {
                                const int sees = (st.lists(y) >> num) & 1 ? lim - st.first(y) : 0, vis = sees - 4 * quad;
                                if (pass == 1) keys += clampi(sees, 0, 2);
#pragma unroll
                                for (int e = 0; e < 4; e++) {
                                    const float p = e < vis ? pow2(__builtin_fmaf(s[y][e], sl2, -lse2)) : 0.f;
                                    if (pass == 0) with_dp += p * d[y][e];
                                    if (pass == 0 || sizeof(T) == 4) total += p;
                                    s[y][e] = p * (d[y][e] - delta) * G.scale;
                                }
                            }
                            if (pass == 1) {
                                const Frag<T> pf = frag_pack<T>(s[0], s[1]);
                                const Columns<T, DP> c(kt[buf], 0, quad, col);
                                if constexpr (sizeof(T) == 2) {
                                    pipelined<Frag<T>, E, 4, 2>([&](int i) { return c.frag(i); },
                                                                [&](int i, const Frag<T> &f) { o[i] = mma(f, pf, o[i]); });
                                } else {
#pragma unroll
                                    for (int j = 0; j < E; j++) o[j] = mma(c.frag(j), pf, o[j]);
                                }
                            }
                        }
                        st = next;
                        __syncthreads();
                    }
                    if (pass == 0) {
                        const float w = quads_sum(with_dp), l = quads_sum(total);
                        delta = (l > 0.f ? w / l : 0.f) - through_lse();
                        total = 0.f;
                    }
                }
            }
            // A value that is no number reaches the columns that do not see it as 0 x NaN: then every row by itself.
            float sum = delta;
#pragma unroll
            for (int j = 0; j < E; j++) sum += (o[j][0] + o[j][1]) + (o[j][2] + o[j][3]);
            if ((now & (now - 1)) && __syncthreads_or(!(fabsf(sum) < INFINITY))) {
                now = todo & -todo;
                continue;
            }
            const Column c1(G, g, slice, per_tile);
            float inv = 1.f;
            if (sizeof(T) == 4) {
                const float l = quads_sum(total);
                inv = l > 0.f ? 1.f / l : 1.f;
            }
            const bool single = keys == 1 && !dlse;
            const int n = wave * per_tile + c1.sub;
            if (c1.live && ((now >> n) & 1)) {
                const long long at = (long long)(t0 + n) * G.heads + c1.head;
                store_row<T, DP>(dq + at * D, o, single ? 0.f : inv, c1.quad, D);
                if (c1.quad == 0) info[at] = RowInfo{lse2, delta, inv, single ? 1.f : 0.f};
            }
            todo &= ~now;
            now = todo & -todo;
        }
        a = z;
    }
}

// ---- the transposed pattern --------------------------------------------------------------------------------------------------
// bits[(mean row * kv_heads + g) * words + t / 64], bit t % 64: query row t lists the block for head g.  One workgroup
// makes the words of 64 rows; of each sequence it writes the words of the blocks that its last row there sees.
__global__ void __launch_bounds__(256)
    k_pattern_bits(const Geometry G, const int *__restrict__ idx, unsigned long long *__restrict__ bits, int words)
{
    __shared__ Union un;
    const int g = (int)(group_id() % G.kv_heads), w = (int)(group_id() / G.kv_heads);
    const int wave = uniform((int)(threadIdx.x >> 6));
    const int t0 = w * 64, t1 = t0 + 64 < G.q_rows ? t0 + 64 : G.q_rows;
    for (int a = t0; a < t1;) {
        Seq sq;
        const int i0 = seq_of_query(G, a, sq);
        if (i0 < 0) {
            a++;
            continue;
        }
        const int z = sq.q_end < t1 ? sq.q_end : t1;
        const int t_mine = t0 + lane_id();
        const int limit = t_mine >= a && t_mine < z ? visible_keys(G, sq, (int)(t_mine - sq.q_base)) : 0;
        const int count = z - a;
        const unsigned long long every = (count < 64 ? (1ULL << count) - 1 : ~0ULL) << (a - t0);
        const int blocks = (read_lane(limit, z - 1 - t0) + G.block - 1) / G.block;
        for (int b0 = 0; b0 < blocks; b0 += kRange) {
            const int nb = blocks - b0 < kRange ? blocks - b0 : kRange;
            union_build(un, G, idx, g, t0, every, limit, b0, nb, wave);
            unsigned long long *p = bits + ((mean_base(G, sq) + b0) * G.kv_heads + g) * words + w;
            for (int x = threadIdx.x; x < nb; x += 256) p[(long long)x * G.kv_heads * words] = un.who[x];
        }
        a = z;
    }
}

// The words that can name rows which see block b of a sequence: k_pattern_bits has written those and no others.
__device__ inline void words_of_block(const Geometry &G, const Seq &sq, int b, int &w0, int &w1)
{
    long long i0 = G.causal ? (long long)b * G.block - (sq.k_len - sq.q_len) : 0;
    long long r0 = sq.q_base + (i0 < 0 ? 0 : i0), r1 = sq.q_base + sq.q_len;
    if (G.cu_q) {
        // the rows that seq_of_query gives the sequence, by the steps of its search: all of them where cu_q ascends
        long long lo = G.cu_q[0], hi = G.cu_q[G.n_seq];
        for (int x = 0, y = G.n_seq; y - x > 1;) {
            const int mid = (x + y) >> 1, c = G.cu_q[mid];
            if (mid <= sq.s) {
                x = mid;
                lo = c > lo ? c : lo;
            } else {
                y = mid;
                hi = c < hi ? c : hi;
            }
        }
        r0 = lo > r0 ? lo : r0;
        r1 = hi < r1 ? hi : r1;
    }
    w0 = (int)(r0 >> 6);
    w1 = r1 > r0 ? (int)((r1 - 1) >> 6) + 1 : w0;
}

// A block's rows are shared out to items of at most `per_item`, all of a block nearly alike.
struct Item {
    int gm, begin, count;     // mean row * kv_heads + head; which of the rows that list the block
    int chunk, chunks, slot;  // of the block's items; where the item's sums go if there are several
};
__global__ void __launch_bounds__(256)
    k_count_rows(const Geometry G, const unsigned long long *__restrict__ bits, int *__restrict__ counts, long long gms, int words)
{
    const long long gm = (long long)group_id() * 4 + (threadIdx.x >> 6);
    if (gm >= gms) return;
    Seq sq;
    int b, n = 0, w0, w1;
    if (!block_of_mean_row(G, gm / G.kv_heads, sq, b)) {
        if (lane_id() == 0) counts[gm] = -1;
        return;
    }
    words_of_block(G, sq, b, w0, w1);
    for (int w = w0 + lane_id(); w < w1; w += 64) n += __popcll(bits[gm * words + w]);
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) n += __shfl_xor(n, d);
    if (lane_id() == 0) counts[gm] = n;
}
__global__ void __launch_bounds__(1024)
    k_plan_items(const int *__restrict__ counts, long long gms, int per_item, Item *__restrict__ items, int *__restrict__ n_items)
{
    __shared__ int sums[2][16];
    const int lane = lane_id(), wave = (int)(threadIdx.x >> 6);
    int base = 0, slots = 0;
    for (long long g0 = 0; g0 < gms; g0 += 1024) {
        const long long gm = g0 + threadIdx.x;
        const int rows = gm < gms ? counts[gm] : -1;
        // a block that no row lists is an item too: its gradients are zeros
        const int n = rows < 0 ? 0 : rows <= per_item ? 1 : (rows + per_item - 1) / per_item, m = n > 1 ? n : 0;
        int a = n, c = m;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int x = __shfl_up(a, d), y = __shfl_up(c, d);
            if (lane >= d) {
                a += x;
                c += y;
            }
        }
        if (lane == 63) {
            sums[0][wave] = a;
            sums[1][wave] = c;
        }
        __syncthreads();
        int at = base + a - n, slot = slots + c - m;
        for (int w = 0; w < 16; w++) {
            if (w < wave) {
                at += sums[0][w];
                slot += sums[1][w];
            }
            base += sums[0][w];
            slots += sums[1][w];
        }
        for (int i = 0; i < n; i++) {
            const int x = (int)((long long)rows * i / n), y = (int)((long long)rows * (i + 1) / n);
            items[at + i] = Item{(int)gm, x, y - x, i, n, slot + i};
        }
        __syncthreads();
    }
    if (threadIdx.x == 0) *n_items = base;
}

// ---- dk, dv -------------------------------------------------------------------------------------------------------------------
// An item's workgroup owns up to 64 keys of the block: KEYS wavefronts side by side with KW x 16 keys each, as the columns of their
// products, and ROWS of them one behind the other, each with its own 32 of the (query, head) pairs that list the block.
// The pairs' rows of q and dout go through LDS (by rows for S = Q K^T and dP = dO V^T, transposed for dK^T = Q^T dS and
// dV^T = dO^T P), fetched while S and dP of the 32 before are computed (the compiler waits for them before the transposed reads).  Bound by what
// LDS delivers: the more keys a wavefront, the fewer reads a product.
// 4096 rows of 32 query and 8 key heads of 128, 16 blocks of 64 each, bf16: 231 us, and 22 for the join of the shared-out blocks' sums; the
// transposed pattern takes 5 us, counting and planning 5 each.  1501 fp32 rows of 6 and 2 heads of 96, 12 blocks of 16 each: 95 and 10 us.
constexpr int kItems = 1024;
constexpr int kListed = 1024;
template <class T, int DP, int KW, int KEYS, int ROWS> struct Dkv {
    static constexpr int KS = DP / 32, E = DP / 16, kThreads = 64 * KEYS * ROWS, kStep = 32 * ROWS;
    static constexpr int kPieces = Tile<T, DP>::kPieces, kTile = kStep * kPieces;
    static constexpr int kDump = KW * 2 * E;  // sums a lane, in fours
    static constexpr int kWaves = DP * sizeof(T) > 256 ? 1 : KW == 1 && kTile <= 512 ? 3 : kTile <= 1024 ? 2 : 1;  // a SIMD: what the sums and the tiles leave room for
    struct Sums {
        f32x4 k[KW][E], v[KW][E];
        __device__ inline f32x4 &at(int i) { return i < KW * E ? k[i / E][i % E] : v[(i - KW * E) / E][i % E]; }
    };
    static __device__ inline void store(const Geometry &G, Sums &a, const Seq &sq, int b, int g, int part, int kw, T *dk, T *dv)
    {
        const int lane = opaque(lane_id()), col = lane & 15, quad = lane >> 4;
#pragma unroll
        for (int x = 0; x < KW; x++) {
            const int key = b * G.block + part * 64 + (kw * KW + x) * 16 + col;
            if (key >= sq.k_len) continue;
            const long long at = ((sq.k_base + key) * G.kv_heads + g) * G.head_dim;
            store_row<T, DP>(dk + at, a.k[x], 1.f, quad, G.head_dim);
            store_row<T, DP>(dv + at, a.v[x], 1.f, quad, G.head_dim);
        }
    }
};

template <class T, int DP, int KW, int KEYS, int ROWS>
__global__ void __launch_bounds__(64 * KEYS * ROWS, (Dkv<T, DP, KW, KEYS, ROWS>::kWaves))
    k_attend_dkv(const Geometry G, const T *__restrict__ q, const T *__restrict__ k, const T *__restrict__ v, const T *__restrict__ dout,
                 const RowInfo *__restrict__ rinfo, const unsigned long long *__restrict__ bits, const Item *__restrict__ items,
                 const int *__restrict__ n_items, f32x4 *__restrict__ slots, T *__restrict__ dk, T *__restrict__ dv, int words, int parts,
                 unsigned group_inv)
{
    using C = Dkv<T, DP, KW, KEYS, ROWS>;
    constexpr int KS = C::KS, E = C::E, kThreads = C::kThreads, kStep = C::kStep, kPieces = C::kPieces;
    __shared__ u32x4 tiles[4 * C::kTile];
    __shared__ int list[kListed];
    __shared__ int listed, passed;
    __shared__ long long still;
    __shared__ __align__(16) float s_lse2[2][kStep], s_delta[2][kStep], s_inv[2][kStep];
    __shared__ __align__(16) int s_limit[2][kStep];
    const int tid = (int)threadIdx.x, lane = lane_id(), col = lane & 15, quad = lane >> 4;
    const int wave = uniform(tid >> 6), kw = wave % KEYS, rw = wave / KEYS;
    const auto qt = [&](int buf) { return tiles + buf * C::kTile; };
    const auto gt = [&](int buf) { return tiles + (2 + buf) * C::kTile; };
    const int part = (int)(group_id() % parts);
    Item it{(int)(group_id() / parts), 0, 0x7fffffff, 0, 1, 0};
    if (items) {
        if (it.gm >= *n_items) return;
        it = items[it.gm];
    }
    const int g = it.gm % G.kv_heads;
    Seq sq;
    int b;
    if (!block_of_mean_row(G, it.gm / G.kv_heads, sq, b)) return;
    const int D = G.head_dim;
    const int key0 = b * G.block + part * 64 + kw * KW * 16 + col;  // inside the sequence; the wavefront's other keys are 16 further
    if (b * G.block + part * 64 >= sq.k_len) return;
    Frag<T> kf[KW][KS], vf[KW][KS];
#pragma unroll
    for (int x = 0; x < KW; x++) {
        const bool mine = key0 + 16 * x < sq.k_len;
        const long long r = sq.k_base + (mine ? key0 + 16 * x : b * G.block);
        row_frags<T, KS, false>(kf[x], k + r * G.k_row + (long long)g * G.k_head, quad, D, mine);
        row_frags<T, KS, false>(vf[x], v + r * G.v_row + (long long)g * G.v_head, quad, D, mine);
    }
    typename C::Sums a;
#pragma unroll
    for (int x = 0; x < KW; x++)
#pragma unroll
        for (int j = 0; j < E; j++) a.k[x][j] = a.v[x][j] = f32x4{0, 0, 0, 0};
    const float sl2 = G.scale * kLog2e;
    const int keys_end = sq.k_len < b * G.block + part * 64 + 64 ? sq.k_len : b * G.block + part * 64 + 64;
    const unsigned long long *mybits = bits + (long long)it.gm * words;
    int w0, w1;
    words_of_block(G, sq, b, w0, w1);
    long long skip = it.begin, left = it.count;  // rows of the earlier items, rows of this one
    for (int w = w0; w < w1 && left > 0;) {
        // up to kListed rows of the item: 64 words at a time
        __syncthreads();
        if (wave == 0) {
            const int lane = opaque(lane_id());
            int have = 0, ww = w;
            long long sk = skip;
            const long long most = left < kListed ? left : kListed;
            while (ww < w1 && have < most) {
                unsigned long long m = ww + lane < w1 ? mybits[ww + lane] : 0;
                const int n = __popcll(m);
                int sum = n;
#pragma unroll
                for (int d = 1; d < 64; d <<= 1) {
                    const int o = pull(sum, lane - d);
                    if (lane >= d) sum += o;
                }
                // words are taken whole: as many as fit
                const bool fits = have + (sum - sk > 0 ? sum - sk : 0) <= kListed;
                const int taken = __popcll(__ballot(fits && ww + lane < w1));
                if (taken == 0) break;
                long long at = (long long)have + sum - n - sk;  // place of the word's first row, negative where an earlier item has it
                const int t0 = (ww + lane) * 64;
                if (lane < taken)
                    while (m) {
                        if (at >= 0 && at < most) list[at] = t0 + __builtin_ctzll(m);
                        at++;
                        m &= m - 1;
                    }
                const int got = read_lane(sum, taken - 1);
                const long long fresh = got - sk;
                sk = fresh < 0 ? -fresh : 0;
                have += fresh > 0 ? (int)fresh : 0;
                ww += taken;
            }
            if (lane == 0) {
                listed = have < most ? have : (int)most;
                passed = ww;
                still = sk;
            }
        }
        __syncthreads();
        const int n = uniform(listed);
        skip = (long long)uniform64((unsigned long long)still);
        w = uniform(passed);
        left -= n;
        const int rows = n * G.group, steps = (rows + kStep - 1) / kStep;
        // row r of the batch: token list[r / group], head r % group
        auto token_of = [&](int r) { return group_inv ? (int)__umulhi((unsigned)r, group_inv) : r; };
        // what there is to know about a row is asked for before its tiles and put into LDS a step later: nothing waits for it
        RowInfo ri;
        int lim;
        auto ask = [&](int step) {
            const int o = opaque(tid), rr = step * kStep + o;
            ri = RowInfo{INFINITY, 0.f, 1.f, 0.f};
            lim = 0;  // of a row with a single key: negative in LDS
            if (o < kStep && rr < rows) {
                const int ti = token_of(rr);
                const long long t = list[ti];
                ri = rinfo[t * G.heads + g * G.group + (rr - ti * G.group)];
                lim = visible_keys(G, sq, (int)(t - sq.q_base));
            }
        };
        auto tell = [&](int buf) {
            const int o = opaque(tid);
            if (o < kStep) {
                s_lse2[buf][o] = ri.lse2;
                s_delta[buf][o] = ri.delta * G.scale;
                if (sizeof(T) == 4) s_inv[buf][o] = ri.inv;
                s_limit[buf][o] = ri.single != 0.f ? -lim : lim;
            }
        };
        auto prepare = [&](int step, int buf) {
            const int o = opaque(tid);
            const int r0 = step * kStep;
            // (asking for whole tiles without the choice: 228 against 240 us)
            const bool whole = D == DP && r0 + kStep <= rows;
#pragma unroll
            for (int i = 0; i < C::kTile / kThreads; i++) {
                const int x = i * kThreads + o, r = x / kPieces, rr = r0 + r;
                const int c = ((x % kPieces) ^ (r & Tile<T, DP>::kSwizzle)) * Tile<T, DP>::kPer;
                const bool in = rr < rows;
                const int ti = token_of(in ? rr : 0), hh = g * G.group + ((in ? rr : 0) - ti * G.group);
                const long long t = list[ti];
                const T *pq = q + t * G.q_row + (long long)hh * G.q_head + c, *pg = dout + (t * G.heads + hh) * D + c;
                const int to = i * kThreads + uniform(o & ~63);
                if (whole) {
                    fetch(qt(buf) + to, pq, true);
                    fetch(gt(buf) + to, pg, true);
                } else {
                    fetch(qt(buf) + to, pq, in && c < D);
                    fetch(gt(buf) + to, pg, in && c < D);
                }
            }
        };
        if (steps > 0) {
            ask(0);
            prepare(0, 0);
            tell(0);
        }
        __syncthreads();
        for (int step = 0; step < steps; step++) {
            const int buf = step & 1;
            if (step + 1 < steps) {
                ask(step + 1);
                prepare(step + 1, buf ^ 1);
            }
            const int base = 32 * rw;
            if (step * kStep + base < rows) {
                Frag<T> pf[KW], df[KW];
                // rows ascend, and so do the keys they see: the first row sees the fewest (rows that are not there see none, and one with a single
                // key, the block's first, comes first too unless the block has no other)
                const int fewest = uniform(s_limit[buf][base]), last = uniform(s_limit[buf][base + 31]);
                const bool all = fewest >= keys_end && last >= keys_end && keys_end > b * G.block + 1;
#pragma unroll
                for (int y = 0; y < 2; y++) {
                    f32x4 s[KW], ds[KW];
#pragma unroll
                    for (int x = 0; x < KW; x++) s[x] = ds[x] = f32x4{0, 0, 0, 0};
                    pipelined<Frag<T>, 2 * KS, 4, 2>(
                        [&](int i) { return tile_frag<T, DP>(i < KS ? qt(buf) : gt(buf), base + 16 * y + col, i % KS, quad); },
                        [&](int i, const Frag<T> &f) {
#pragma unroll
                            for (int x = 0; x < KW; x++) {
                                if (i < KS) s[x] = mma(f, kf[x][i % KS], s[x]);
                                else ds[x] = mma(f, vf[x][i % KS], ds[x]);
                            }
                        });
                    const int r = base + 16 * y + 4 * quad;
                    const f32x4 l2 = *(const f32x4 *)&s_lse2[buf][r], de = *(const f32x4 *)&s_delta[buf][r];
                    f32x4 iv = f32x4{1.f, 1.f, 1.f, 1.f};
                    if (sizeof(T) == 4) iv = *(const f32x4 *)&s_inv[buf][r];
#pragma unroll
                    for (int x = 0; x < KW; x++)
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            float p = pow2(__builtin_fmaf(s[x][e], sl2, -l2[e]));
                            if (sizeof(T) == 4) p *= iv[e];
                            s[x][e] = p;
                            ds[x][e] = p * __builtin_fmaf(ds[x][e], G.scale, -de[e]);
                        }
                    if (!all) {
                        typedef __attribute__((ext_vector_type(4))) int i32x4;
                        const i32x4 li = *(const i32x4 *)&s_limit[buf][r];
#pragma unroll
                        for (int x = 0; x < KW; x++)
#pragma unroll
                            for (int e = 0; e < 4; e++) {
                                const bool single = li[e] < 0, on = key0 + 16 * x < (single ? -li[e] : li[e]);
                                s[x][e] = on ? s[x][e] : 0.f;
                                ds[x][e] = on ? (single ? 0.f * ds[x][e] : ds[x][e]) : 0.f;  // what is no number stays so
                            }
                    }
#pragma unroll
                    for (int x = 0; x < KW; x++) {
                        frag_half(pf[x], y, s[x]);
                        frag_half(df[x], y, ds[x]);
                    }
                }
                if constexpr (sizeof(T) == 2) {
                    pipelined<Frag<T>, 2 * E, 4, 2>(
                        [&](int i) { return Columns<T, DP>(i < E ? gt(buf) : qt(buf), 2 * rw, quad, col).frag(i % E); },
                        [&](int i, const Frag<T> &f) {
#pragma unroll
                            for (int x = 0; x < KW; x++) {
                                if (i < E) a.v[x][i % E] = mma(f, pf[x], a.v[x][i % E]);
                                else a.k[x][i % E] = mma(f, df[x], a.k[x][i % E]);
                            }
                        });
                } else {
                    {
                        const Columns<T, DP> c(gt(buf), 2 * rw, quad, col);
#pragma unroll
                        for (int j = 0; j < E; j++)
#pragma unroll
                            for (int x = 0; x < KW; x++) a.v[x][j] = mma(c.frag(j), pf[x], a.v[x][j]);
                    }
                    {
                        const Columns<T, DP> c(qt(buf), 2 * rw, quad, col);
#pragma unroll
                        for (int j = 0; j < E; j++)
#pragma unroll
                            for (int x = 0; x < KW; x++) a.k[x][j] = mma(c.frag(j), df[x], a.k[x][j]);
                    }
                }
            }
            if (step + 1 < steps) tell(buf ^ 1);
            __syncthreads();
        }
    }
    // the wavefronts with other rows: added up in their order
    if constexpr (ROWS > 1) {
        f32x4 *ex = (f32x4 *)tiles;
        constexpr int kHalf = C::kDump / 2;  // dk's sums, then dv's
        static_assert((ROWS - 1) * KEYS * kHalf * 64 * 16 <= (int)sizeof(tiles), "the exchange fits the tiles");
#pragma unroll
        for (int h = 0; h < 2; h++) {
            __syncthreads();
            if (rw > 0) {
#pragma unroll
                for (int i = 0; i < kHalf; i++) ex[(((rw - 1) * KEYS + kw) * kHalf + i) * 64 + lane] = a.at(h * kHalf + i);
            }
            __syncthreads();
            if (rw == 0) {
#pragma unroll
                for (int w = 0; w < ROWS - 1; w++)
#pragma unroll
                    for (int i = 0; i < kHalf; i++) a.at(h * kHalf + i) += ex[((w * KEYS + kw) * kHalf + i) * 64 + lane];
            }
        }
        if (rw > 0) return;
    }
    if (it.chunks > 1) {
        f32x4 *p = slots + (((long long)it.slot * parts + part) * KEYS + kw) * C::kDump * 64 + lane;
#pragma unroll
        for (int i = 0; i < C::kDump; i++) p[i * 64] = a.at(i);
    } else {
        C::store(G, a, sq, b, g, part, kw, dk, dv);
    }
}

// Blocks of several items: the items' sums, added in their order.
template <class T, int DP, int KW, int KEYS, int ROWS>
__global__ void __launch_bounds__(64 * KEYS)
    k_join_dkv(const Geometry G, const Item *__restrict__ items, const int *__restrict__ n_items, const f32x4 *__restrict__ slots, T *__restrict__ dk,
               T *__restrict__ dv, int parts)
{
    using C = Dkv<T, DP, KW, KEYS, ROWS>;
    const int part = (int)(group_id() % parts), i = (int)(group_id() / parts);
    if (i >= *n_items) return;
    const Item it = items[i];
    if (it.chunks < 2 || it.chunk != 0) return;
    Seq sq;
    int b;
    if (!block_of_mean_row(G, it.gm / G.kv_heads, sq, b) || b * G.block + part * 64 >= sq.k_len) return;
    const int kw = uniform((int)(threadIdx.x >> 6)), lane = lane_id();
    typename C::Sums a;
    const f32x4 *p = slots + (((long long)it.slot * parts + part) * KEYS + kw) * C::kDump * 64 + lane;
    const long long apart = (long long)parts * KEYS * C::kDump * 64;
#pragma unroll
    for (int x = 0; x < C::kDump; x++) a.at(x) = p[x * 64];
    // a few items' sums are on their way at a time
    constexpr int kAhead = C::kDump <= 16 ? 4 : 2;
    for (int c = 1; c < it.chunks; c += kAhead) {
        f32x4 w[kAhead][C::kDump];
#pragma unroll
        for (int u = 0; u < kAhead; u++)
#pragma unroll
            for (int x = 0; x < C::kDump; x++) w[u][x] = c + u < it.chunks ? p[(c + u) * apart + x * 64] : f32x4{0, 0, 0, 0};
#pragma unroll
        for (int u = 0; u < kAhead; u++)
#pragma unroll
            for (int x = 0; x < C::kDump; x++) a.at(x) += w[u][x];
    }
    C::store(G, a, sq, b, it.gm % G.kv_heads, part, kw, dk, dv);
}

// What the backward pass keeps in the workspace.
struct BwdSpace {
    long long gms, max_items, info_at, bits_at, counts_at, items_at, slots_at, total;
    int words, per_item, parts;
    bool shared_out;  // some block may have more rows than an item
};
static BwdSpace bwd_space(const Geometry &G)
{
    BwdSpace s;
    const auto up = [](long long x) { return ceil_div(x, 256) * 256; };
    s.gms = (G.cu_k ? G.k_rows / G.block + G.n_seq : (long long)G.blocks_each * G.n_seq) * G.kv_heads;
    s.words = (int)ceil_div(G.q_rows, 64);
    s.parts = G.block > 64 ? G.block / 64 : 1;
    // about 1024 items besides the blocks' own, of at least 64 rows (4096 rows of 32/8 heads whose first block all list, the whole gradient with
    // 512, 1024, 2048: 395, 354, 376 us; 1024 rows: 148, 143, 164; 16384 rows of 8/2 heads: 441, 428, 485)
    const long long listed = (long long)G.q_rows * G.kv_heads * G.width;
    s.per_item = 64;
    while (listed / s.per_item > kItems) s.per_item *= 2;
    s.shared_out = G.q_rows > s.per_item;
    s.max_items = s.gms + (s.shared_out ? listed / s.per_item : 0);
    // a block with n > per_item rows has at most 2 n / per_item items
    const long long keep = s.shared_out ? 2 * (listed / s.per_item + 1) : 0;
    const int dims = G.head_dim <= 64 ? 64 : G.head_dim <= 128 ? 128 : 256;
    s.info_at = 0;
    s.bits_at = up((long long)G.q_rows * G.heads * (long long)sizeof(RowInfo));
    s.counts_at = s.bits_at + up(8 * s.gms * s.words);
    s.items_at = s.counts_at + (s.shared_out ? up(4 * (s.gms + 1)) : 0);
    s.slots_at = s.items_at + (s.shared_out ? up((long long)sizeof(Item) * s.max_items) : 0);
    s.total = s.slots_at + keep * G.block * dims * 2 * 4;
    return s;
}

template <class T, int DP, int KW, int KEYS, int ROWS>
static void launch_dkv(const Geometry &G, const void *q, const void *k, const void *v, const void *dout, void *dk, void *dv, char *ws,
                       const BwdSpace &sp, hipStream_t st)
{
    const RowInfo *info = (const RowInfo *)(ws + sp.info_at);
    const unsigned long long *bits = (const unsigned long long *)(ws + sp.bits_at);
    const Item *items = sp.shared_out ? (const Item *)(ws + sp.items_at) : nullptr;
    const int *n_items = (const int *)(ws + sp.counts_at) + sp.gms;
    f32x4 *slots = (f32x4 *)(ws + sp.slots_at);
    // floor(r * inv / 2^32) = r / group for r < kListed * group <= 2^20: inv is off by less than group / 2^32 of 1 / group
    const unsigned inv = G.group == 1 ? 0 : (unsigned)((0x100000000ULL + G.group - 1) / G.group);
    launch((k_attend_dkv<T, DP, KW, KEYS, ROWS>), groups(sp.max_items * sp.parts), dim3(64 * KEYS * ROWS), 0, st, G,
                       (const T *)q, (const T *)k, (const T *)v, (const T *)dout, info, bits, items, n_items, slots, (T *)dk, (T *)dv, sp.words,
                       sp.parts, inv);
    if (sp.shared_out)
        launch((k_join_dkv<T, DP, KW, KEYS, ROWS>), groups(sp.max_items * sp.parts), dim3(64 * KEYS), 0, st, G, items, n_items,
                           slots, (T *)dk, (T *)dv, sp.parts);
}

template <class T, int DP>
static void launch_bwd(const Geometry &G, const void *q, const void *k, const void *v, const int *idx, const void *out, const float *lse,
                       const void *dout, const float *dlse, void *dq, void *dk, void *dv, char *ws, const BwdSpace &sp, hipStream_t st)
{
    RowInfo *info = (RowInfo *)(ws + sp.info_at);
    unsigned long long *bits = (unsigned long long *)(ws + sp.bits_at);
    const int slices = (int)ceil_div(G.group, 16);
    if (G.q_rows > 0) {
        const int per_tile = G.group < 16 ? 16 / G.group : 1;
#define NSP_GO(WIDE)                                                                                                                     \
    launch((k_attend_dq<T, DP, WIDE>), groups(ceil_div(G.q_rows, 4 * per_tile) * slices * G.kv_heads), \
                       dim3(256), 0, st, G, (const T *)q, (const T *)k, (const T *)v, idx, (const T *)out, lse, (const T *)dout, dlse,       \
                       (T *)dq, info, slices, per_tile)
        if (G.block >= 32) NSP_GO(true); else NSP_GO(false);
#undef NSP_GO
        if (sp.gms > 0) {
            launch(k_pattern_bits, groups((long long)sp.words * G.kv_heads), dim3(256), 0, st, G, idx, bits, sp.words);
            if (sp.shared_out) {
                int *counts = (int *)(ws + sp.counts_at);
                launch(k_count_rows, groups(ceil_div(sp.gms, 4)), dim3(256), 0, st, G, bits, counts, sp.gms, sp.words);
                launch(k_plan_items, dim3(1), dim3(1024), 0, st, counts, sp.gms, sp.per_item, (Item *)(ws + sp.items_at), counts + sp.gms);
            }
        }
    }
    if (sp.gms == 0) return;
    // Keys a wavefront, then wavefronts over the keys x over the rows, as the sums' registers and the tiles' LDS allow.
    constexpr int kWide = sizeof(T) == 2 && DP <= 64 ? 2 : 1;
    constexpr int kMost = 128 * 1024 / (4 * 32 * DP * (int)sizeof(T));  // wavefronts over the rows that 128 KB hold tiles for
    constexpr int kKw2 = kWide < 2 ? 1 : 2, kKeys2 = 2 / kKw2, kKeys4 = 4 / kWide;
    constexpr int kRows1 = kMost < 4 ? kMost : 4, kRows2 = kMost < 4 / kKeys2 ? kMost : 4 / kKeys2, kRows4 = kMost < 4 / kKeys4 ? kMost : 4 / kKeys4;
    if (G.block == 16)
        launch_dkv<T, DP, 1, 1, kRows1>(G, q, k, v, dout, dk, dv, ws, sp, st);
    else if (G.block == 32)
        launch_dkv<T, DP, kKw2, kKeys2, kRows2>(G, q, k, v, dout, dk, dv, ws, sp, st);
    else
        launch_dkv<T, DP, kWide, kKeys4, kRows4>(G, q, k, v, dout, dk, dv, ws, sp, st);
}

}  // namespace lm
}  // namespace nsp

extern "C" {

long long nsparse_lm_block_attention_bwd_workspace(const nsparse_lm_attn *a)
{
    using namespace nsp::lm;
    clear_error();
    Geometry G;
    if (int rc = geometry(a, false, false, &G)) return rc;
    if (G.page_size > 0) return fail(NSPARSE_LM_EARG, "block_attention_bwd: not for paged caches");
    return bwd_space(G).total;
}

int nsparse_lm_block_attention_lse_bwd(const nsparse_lm_attn *a, const void *q, const void *k, const void *v, const int *idx, const void *out,
                                       const float *lse, const void *dout, const float *dlse, void *dq, void *dk, void *dv, void *workspace,
                                       long long workspace_bytes, void *stream)
{
    using namespace nsp::lm;
    clear_error();
    Geometry G;
    if (int rc = geometry(a, true, true, &G)) return rc;
    if (G.page_size > 0) return fail(NSPARSE_LM_EARG, "block_attention_bwd: not for paged caches");
    const BwdSpace sp = bwd_space(G);
    if (sp.max_items * sp.parts > kMostGroups) return fail(NSPARSE_LM_EARG, "block_attention_bwd: blocks x heads out of range");
    if ((G.q_rows > 0 && (!q || !idx || !out || !lse || !dout || !dq)) || (G.k_rows > 0 && (!k || !v || !dk || !dv)))
        return fail(NSPARSE_LM_EARG, "block_attention_bwd: a required pointer is NULL");
    if (((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)out | (uintptr_t)dout | (uintptr_t)dq | (uintptr_t)dk | (uintptr_t)dv |
         (uintptr_t)workspace) & 15)
        return fail(NSPARSE_LM_EALIGN, "block_attention_bwd: tensors and workspace begin at multiples of 16 bytes");
    if (sp.total > 0 && (!workspace || workspace_bytes < sp.total))
        return fail(NSPARSE_LM_EWORKSPACE, "block_attention_bwd: workspace smaller than nsparse_lm_block_attention_bwd_workspace() says");
    hipStream_t st = (hipStream_t)stream;
    char *ws = (char *)workspace;
#define NSP_DIM(T)                                                                                                  \
    if (G.head_dim <= 64) launch_bwd<T, 64>(G, q, k, v, idx, out, lse, dout, dlse, dq, dk, dv, ws, sp, st);         \
    else if (G.head_dim <= 128) launch_bwd<T, 128>(G, q, k, v, idx, out, lse, dout, dlse, dq, dk, dv, ws, sp, st);  \
    else launch_bwd<T, 256>(G, q, k, v, idx, out, lse, dout, dlse, dq, dk, dv, ws, sp, st)
    if (a->dtype == NSPARSE_LM_BF16) { NSP_DIM(__bf16); }
    else if (a->dtype == NSPARSE_LM_F16) { NSP_DIM(_Float16); }
    else { NSP_DIM(float); }
#undef NSP_DIM
    return launched("block_attention_bwd");
}

int nsparse_lm_block_attention_bwd(const nsparse_lm_attn *a, const void *q, const void *k, const void *v, const int *idx, const void *out,
                                   const float *lse, const void *dout, void *dq, void *dk, void *dv, void *workspace,
                                   long long workspace_bytes, void *stream)
{
    return nsparse_lm_block_attention_lse_bwd(a, q, k, v, idx, out, lse, dout, nullptr, dq, dk, dv, workspace, workspace_bytes, stream);
}
}
