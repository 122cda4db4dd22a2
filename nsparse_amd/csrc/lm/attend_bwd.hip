// attend_bwd.hip -- gradient of attention over the listed blocks of keys.
//
//   p = exp(s - lse), delta = dout . out, ds = p (dout . v - delta)
//   dq = scale sum_j ds_j k_j          over the keys that the query's row lists: the pattern, one wavefront a row
//   dk = scale sum_t ds_t q_t, dv = sum_t p_t dout_t    over the queries that list the key's block: the transposed pattern
//
// The transposed pattern is a bitmap: for every key head and block one bit a query row, built by 64 rows a workgroup in
// LDS and written as whole words, so it needs no counting, no sort and no atomics on memory, and the order of
// the sums in dk and dv is the order of the rows, whatever the timing.  p and scale * ds are rounded to the inputs' type for the second
// products (with the scale, so that half precision overflows no sooner than the gradients themselves do).
#include "attend.h"

namespace nsp {
namespace lm {

// ---- dq (and delta) ----------------------------------------------------------------------------------------------------
// As the forward for prompts (attend_fwd.hip): the workgroup's rows are the columns of its products, the union of their blocks goes
// through LDS.  S^T = K Q^T and dP^T = V dO^T read K and V by rows, dQ^T = K^T dS^T reads K transposed.
// delta comes from the output as the forward rounded it.  That rounding matters where few keys share the weight, so workgroups with
// at most kExact keys in their union walk twice and take delta = sum p (dout . v) from the first walk.  In single precision the
// probabilities are divided by their sum, which takes the rounding of the log-sum-exp out of them.
constexpr int kExact = 256;
struct RowInfo {  // of a query row and head, for dk and dv
    float lse2, delta, inv;
    float pad;
};
template <class T, int DP, int NT, int NG, bool WIDE>
__global__ void __launch_bounds__(256, DP * sizeof(T) <= 256 ? 2 : 1)
    k_attend_dq(const Geometry G, const T *__restrict__ q, const T *__restrict__ k, const T *__restrict__ v, const int *__restrict__ idx,
                const T *__restrict__ out, const float *__restrict__ lse, const T *__restrict__ dout, T *__restrict__ dq,
                RowInfo *__restrict__ info, int slices, int per_tile)
{
    constexpr int KS = DP / 32, E = DP / 16, kTile = NG * 16 * Tile<T, DP>::kPieces;
    __shared__ u32x4 kt[2][kTile], vt[2][kTile];
    __shared__ Union un;
    const int wave = uniform((int)(threadIdx.x >> 6));
    const int g = (int)(blockIdx.x % G.kv_heads);
    const int rest = (int)(blockIdx.x / G.kv_heads);
    const int slice = rest % slices;
    const int per_wave = NT * per_tile;  // rows a wavefront
    const int t0 = (rest / slices) * 4 * per_wave;
    const int t1 = t0 + 4 * per_wave < G.q_rows ? t0 + 4 * per_wave : G.q_rows;
    const int D = G.head_dim;
    const float sl2 = G.scale * kLog2e;

    for (int a = t0; a < t1;) {
        Seq sq;
        const int i0 = seq_of_query(G, a, sq);
        if (i0 < 0) {
            a++;
            continue;
        }
        const int z = sq.q_base + sq.q_len < t1 ? (int)(sq.q_base + sq.q_len) : t1;
        const Column c0(G, g, slice, per_tile);
        const int col = c0.col, quad = c0.quad;
        // lane i's row for the walk; a column's row is number (wave * NT + x) * per_tile + Column::sub
        const int t_mine = t0 + opaque(lane_id());
        const int limit = t_mine >= a && t_mine < z ? visible_keys(G, sq, (int)(t_mine - sq.q_base)) : 0;
        Frag<T> qf[NT][KS], gf[NT][KS];
        int lim[NT], num[NT];
        float lse2[NT], rounded[NT];
#pragma unroll
        for (int x = 0; x < NT; x++) {
            num[x] = (wave * NT + x) * per_tile + c0.sub;
            const bool on = c0.live && t0 + num[x] >= a && t0 + num[x] < z;
            lim[x] = pull(limit, num[x]);
            if (!on) lim[x] = 0;
            const int t = on ? t0 + num[x] : a;
            const long long th = (long long)t * G.heads + c0.head;
            row_frags<T, KS, false>(gf[x], dout + th * D, quad, D, on);
            row_frags<T, KS, false>(qf[x], out + th * D, quad, D, on);
            rounded[x] = 0.f;
#pragma unroll
            for (int w = 0; w < KS; w++) rounded[x] += frag_dot(gf[x][w], qf[x][w]);
            rounded[x] = quads_sum(rounded[x]);
            row_frags<T, KS, false>(qf[x], q + (long long)t * G.q_row + (long long)c0.head * G.q_head, quad, D, on);
            lse2[x] = on ? lse[th] * kLog2e : INFINITY;
        }
        const int count = z - a;
        const unsigned long long every = (count < 64 ? (1ULL << count) - 1 : ~0ULL) << (a - t0);
        unsigned long long todo = every, now = every;
        while (todo) {
            f32x4 o[NT][E];
            float total[NT], with_dp[NT], delta[NT];
#pragma unroll
            for (int x = 0; x < NT; x++) {
                total[x] = with_dp[x] = 0.f;
                delta[x] = rounded[x];
#pragma unroll
                for (int j = 0; j < E; j++) o[x][j] = f32x4{0, 0, 0, 0};
            }
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
                        const bool use = (st.any >> (wave * NT * per_tile)) & (NT * per_tile < 64 ? (1ULL << (NT * per_tile)) - 1 : ~0ULL);
                        if (use) {
#pragma unroll
                            for (int y2 = 0; y2 < NG; y2 += 2) {
                                Frag<T> pf[NT];
                                f32x4 s[NT][2], d[NT][2];
#pragma unroll
                                for (int x = 0; x < NT; x++) s[x][0] = s[x][1] = d[x][0] = d[x][1] = f32x4{0, 0, 0, 0};
                                pipelined<Frag<T>, 4 * KS, 4, 2>(
                                    [&](int i) {
                                        const int r = 16 * (y2 + (i / KS & 1)) + col;
                                        return tile_frag<T, DP>(i < 2 * KS ? kt[buf] : vt[buf], r, i % KS, quad);
                                    },
                                    [&](int i, const Frag<T> &f) {
                                        const int y = i / KS & 1;
#pragma unroll
                                        for (int x = 0; x < NT; x++) {
                                            if (i < 2 * KS) s[x][y] = mma(f, qf[x][i % KS], s[x][y]);
                                            else d[x][y] = mma(f, gf[x][i % KS], d[x][y]);
                                        }
                                    });
#pragma unroll
                                for (int x = 0; x < NT; x++) {
#pragma unroll
                                    for (int y = 0; y < 2; y++) {
                                        const bool on = (st.lists(y2 + y) >> num[x]) & 1;
                                        const int vis = on ? lim[x] - st.first(y2 + y) - 4 * quad : 0;
#pragma unroll
                                        for (int e = 0; e < 4; e++) {
                                            const float p = e < vis ? pow2(__builtin_fmaf(s[x][y][e], sl2, -lse2[x])) : 0.f;
                                            if (pass == 0) with_dp[x] += p * d[x][y][e];
                                            if (pass == 0 || sizeof(T) == 4) total[x] += p;
                                            s[x][y][e] = p * (d[x][y][e] - delta[x]) * G.scale;
                                        }
                                    }
                                    pf[x] = frag_pack<T>(s[x][0], s[x][1]);
                                }
                                if (pass == 0) continue;
                                if constexpr (sizeof(T) == 2) {
                                    pipelined<Frag<T>, E, 4, 2>([&](int i) { return Columns<T, DP>(kt[buf], y2, quad, col).frag(i); },
                                                                [&](int i, const Frag<T> &f) {
#pragma unroll
                                                                    for (int x = 0; x < NT; x++) o[x][i] = mma(f, pf[x], o[x][i]);
                                                                });
                                } else {
                                    const Columns<T, DP> c(kt[buf], y2, quad, col);
#pragma unroll
                                    for (int j = 0; j < E; j++) {
                                        const Frag<T> f = c.frag(j);
#pragma unroll
                                        for (int x = 0; x < NT; x++) o[x][j] = mma(f, pf[x], o[x][j]);
                                    }
                                }
                            }
                        }
                        st = next;
                        __syncthreads();
                    }
                    if (pass == 0) {
#pragma unroll
                        for (int x = 0; x < NT; x++) {
                            const float w = quads_sum(with_dp[x]), l = quads_sum(total[x]);
                            delta[x] = l > 0.f ? w / l : 0.f;
                            total[x] = 0.f;
                        }
                    }
                }
            }
            // A value that is no number reaches the columns that do not see it as 0 x NaN: then every row by itself.
            bool bad = false;
#pragma unroll
            for (int x = 0; x < NT; x++) {
                float t = delta[x];
#pragma unroll
                for (int j = 0; j < E; j++) t += (o[x][j][0] + o[x][j][1]) + (o[x][j][2] + o[x][j][3]);
                bad = bad || !(fabsf(t) < INFINITY);
            }
            if ((now & (now - 1)) && __syncthreads_or(bad)) {
                now = todo & -todo;
                continue;
            }
            const Column c1(G, g, slice, per_tile);
#pragma unroll
            for (int x = 0; x < NT; x++) {
                float inv = 1.f;
                if (sizeof(T) == 4) {
                    const float l = quads_sum(total[x]);
                    inv = l > 0.f ? 1.f / l : 1.f;
                }
                const int n = (wave * NT + x) * per_tile + c1.sub;
                if (!c1.live || !((now >> n) & 1)) continue;
                const long long th = (long long)(t0 + n) * G.heads + c1.head;
                store_row<T, DP>(dq + th * D, o[x], inv, c1.quad, D);
                if (c1.quad == 0) info[th] = RowInfo{lse2[x], delta[x], inv, 0.f};
            }
            todo &= ~now;
            now = todo & -todo;
        }
        a = z;
    }
}

// ---- the transposed pattern --------------------------------------------------------------------------------------------------
// bits[(g * mean_rows + mean row) * words + t / 64], bit t % 64: query row t lists the block for head g.  One workgroup
// makes the words of 64 rows; of each sequence it writes the words of the blocks that its last row there sees.
constexpr int kBitBlocks = 4096;
__global__ void __launch_bounds__(256)
    k_pattern_bits(const Geometry G, const int *__restrict__ idx, unsigned long long *__restrict__ bits, long long mean_rows, int words)
{
    __shared__ unsigned half[2 * kBitBlocks];
    const int g = (int)(blockIdx.x % G.kv_heads), w = (int)(blockIdx.x / G.kv_heads);
    const int wave = threadIdx.x >> 6;
    const int t0 = w * 64, t1 = t0 + 64 < G.q_rows ? t0 + 64 : G.q_rows;
    // the first sequence that reaches into these rows
    int s = 0;
    if (G.cu_q) {
        int hi = G.n_seq;
        while (hi - s > 1) {
            const int mid = (s + hi) >> 1;
            if (G.cu_q[mid] <= t0) s = mid; else hi = mid;
        }
    } else {
        s = t0 / G.q_each;
    }
    for (; s < G.n_seq; s++) {
        const Seq sq = seq_at(G, s);
        if (sq.q_base >= t1) break;
        const int a = sq.q_base > t0 ? (int)sq.q_base : t0;
        const int z = sq.q_base + sq.q_len < t1 ? (int)(sq.q_base + sq.q_len) : t1;
        if (z <= a) continue;
        const int seen_blocks = (visible_keys(G, sq, (int)(z - 1 - sq.q_base)) + G.block - 1) / G.block;
        for (int b0 = 0; b0 < seen_blocks; b0 += kBitBlocks) {
            const int nb = seen_blocks - b0 < kBitBlocks ? seen_blocks - b0 : kBitBlocks;
            for (int x = threadIdx.x; x < 2 * nb; x += 256) half[x] = 0;
            __syncthreads();
            for (int t = a + wave; t < z; t += 4) {
                const int limit = visible_keys(G, sq, (int)(t - sq.q_base));
                const int *row = idx + ((long long)t * G.kv_heads + g) * G.width;
                int seen = -1;
                for (int at = 0; at < G.width; at += 64) {
                    int b;
                    const int n = pattern_chunk(row, at, G.width, (limit + G.block - 1) / G.block, seen, b);
                    if (lane_id() < n && b >= b0 && b < b0 + nb)
                        atomicOr(&half[2 * (b - b0) + ((t - t0) >> 5)], 1u << ((t - t0) & 31));
                }
            }
            __syncthreads();
            unsigned long long *p = bits + ((long long)g * mean_rows + mean_base(G, sq) + b0) * words + w;
            for (int x = threadIdx.x; x < nb; x += 256)
                p[(long long)x * words] = ((unsigned long long)half[2 * x + 1] << 32) | half[2 * x];
            __syncthreads();
        }
    }
}

// ---- dk, dv -------------------------------------------------------------------------------------------------------------------
// One workgroup per (key head, block, 64 of its keys); wavefront x owns sixteen of the keys, as the columns of its products.  The rows
// are the (query, head) pairs that list the block, 32 at a time.
constexpr int kListWords = 64;
template <class T, int DP, bool FULL>
__global__ void __launch_bounds__(256)
    k_attend_dkv(const Geometry G, const T *__restrict__ q, const T *__restrict__ k, const T *__restrict__ v,
                 const T *__restrict__ dout, const RowInfo *__restrict__ rinfo, const unsigned long long *__restrict__ bits, T *__restrict__ dk,
                 T *__restrict__ dv, long long mean_rows, int words, int parts)
{
    constexpr int KS = DP / 32, E = DP / 16;
    __shared__ int list[kListWords * 64];
    __shared__ int listed;
    struct Info {
        long long q_off[32], o_off[32];
        float lse2[32], delta[32], inv[32];
        int limit[32];
    };
    __shared__ Info infos[4];
    const int lane = lane_id(), col = lane & 15, quad = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const int g = (int)(blockIdx.x % G.kv_heads);
    const long long rest = blockIdx.x / G.kv_heads;
    const long long mrow = rest / parts;
    Seq sq;
    int b;
    if (!block_of_mean_row(G, mrow, sq, b)) return;
    const int D = G.head_dim;
    const int key = b * G.block + (int)(rest % parts) * 64 + wave * 16 + col;  // inside the sequence
    const bool mine = key < sq.k_len;
    const long long krow = sq.k_base + (mine ? key : b * G.block);
    Frag<T> kf[KS], vf[KS];
    row_frags<T, KS, FULL>(kf, k + krow * G.k_row + (long long)g * G.k_head, quad, D, mine);
    row_frags<T, KS, FULL>(vf, v + krow * G.v_row + (long long)g * G.v_head, quad, D, mine);
    f32x4 ak[E], av[E];
#pragma unroll
    for (int j = 0; j < E; j++) ak[j] = av[j] = f32x4{0, 0, 0, 0};
    const float sl2 = G.scale * kLog2e;
    Info &in = infos[wave];
    const unsigned long long *mybits = bits + ((long long)g * mean_rows + mrow) * words;
    // the rows that can see the block's first key
    int i0 = G.causal ? b * G.block - (sq.k_len - sq.q_len) : 0;
    if (i0 < 0) i0 = 0;
    const int w0 = (int)((sq.q_base + i0) >> 6), w1 = sq.q_len > i0 ? (int)((sq.q_base + sq.q_len - 1) >> 6) + 1 : w0;
    for (int wb = w0; wb < w1; wb += kListWords) {
        __syncthreads();
        if (wave == 0) {
            unsigned long long m = wb + lane < w1 ? mybits[wb + lane] : 0;
            int at = __popcll(m);
            int sum = at;
#pragma unroll
            for (int d = 1; d < 64; d <<= 1) {
                const int o = __shfl_up(sum, d);
                if (lane >= d) sum += o;
            }
            at = sum - at;
            if (lane == 63) listed = sum;
            const int t0 = (wb + lane) * 64;
            while (m) {
                list[at++] = t0 + __builtin_ctzll(m);
                m &= m - 1;
            }
        }
        __syncthreads();
        const long long rows = (long long)listed * G.group;
        for (long long r0 = 0; r0 < rows; r0 += 32) {
            __builtin_amdgcn_wave_barrier();
            if (lane < 32) {
                const long long r = r0 + lane;
                const bool ok = r < rows;
                const int t = list[ok ? r / G.group : 0], h = g * G.group + (ok ? (int)(r % G.group) : 0);
                const long long th = (long long)t * G.heads + h;
                in.q_off[lane] = (long long)t * G.q_row + (long long)h * G.q_head;
                in.o_off[lane] = th * D;
                const RowInfo ri = rinfo[th];
                in.lse2[lane] = ri.lse2;
                in.delta[lane] = ri.delta;
                in.inv[lane] = ri.inv;
                in.limit[lane] = ok ? visible_keys(G, sq, (int)(t - sq.q_base)) : 0;
            }
            __builtin_amdgcn_wave_barrier();
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            const bool whole = r0 + 32 <= rows;
            f32x4 s[2], ds[2];
#pragma unroll
            for (int y = 0; y < 2; y++) {
                Frag<T> f[KS];
                f32x4 dp = f32x4{0, 0, 0, 0};
                s[y] = f32x4{0, 0, 0, 0};
                row_frags<T, KS, FULL>(f, q + in.q_off[16 * y + col], quad, D, true);
#pragma unroll
                for (int z = 0; z < KS; z++) s[y] = mma(f[z], kf[z], s[y]);
                row_frags<T, KS, FULL>(f, dout + in.o_off[16 * y + col], quad, D, true);
#pragma unroll
                for (int z = 0; z < KS; z++) dp = mma(f[z], vf[z], dp);
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const int r = 16 * y + 4 * quad + e;
                    const bool on = mine && key < in.limit[r];
                    s[y][e] = on ? pow2(__builtin_fmaf(s[y][e], sl2, -in.lse2[r])) : 0.f;
                    if (sizeof(T) == 4) s[y][e] *= in.inv[r];
                    ds[y][e] = on ? s[y][e] * (dp[e] - in.delta[r]) * G.scale : 0.f;
                }
            }
            {
                Rows<T, E> x;
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const int r = (e < 4 ? 0 : 16) + 4 * quad + (e & 3);
                    const T *p = dout + in.o_off[r] + col * E;
                    if constexpr (FULL) rows_load(x, e, p); else rows_load_part(x, e, p, D - col * E);
                    if (!whole && r0 + r >= rows) rows_clear(x, e);
                }
                const Frag<T> pf = frag_pack<T>(s[0], s[1]);
#pragma unroll
                for (int j = 0; j < E; j++) av[j] = mma(rows_column(x, j), pf, av[j]);
            }
            {
                Rows<T, E> x;
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const int r = (e < 4 ? 0 : 16) + 4 * quad + (e & 3);
                    const T *p = q + in.q_off[r] + col * E;
                    if constexpr (FULL) rows_load(x, e, p); else rows_load_part(x, e, p, D - col * E);
                    if (!whole && r0 + r >= rows) rows_clear(x, e);
                }
                const Frag<T> sf = frag_pack<T>(ds[0], ds[1]);
#pragma unroll
                for (int j = 0; j < E; j++) ak[j] = mma(rows_column(x, j), sf, ak[j]);
            }
        }
    }
    if (mine) {
        const long long at = (krow * G.kv_heads + g) * D;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const int d = (4 * quad + e) * E;
            float x[E];
#pragma unroll
            for (int j = 0; j < E; j++) x[j] = av[j][e];
            store_columns<T, E>(dv + at + d, x, D - d);
#pragma unroll
            for (int j = 0; j < E; j++) x[j] = ak[j][e];
            store_columns<T, E>(dk + at + d, x, D - d);
        }
    }
}

struct BwdSpace {
    long long mean_rows, info_bytes, total;
    int words;
};
static BwdSpace bwd_space(const Geometry &G)
{
    BwdSpace s;
    s.mean_rows = G.cu_k ? G.k_rows / G.block + G.n_seq : (long long)G.blocks_each * G.n_seq;
    s.words = (int)ceil_div(G.q_rows, 64);
    s.info_bytes = ceil_div((long long)G.q_rows * G.heads * (long long)sizeof(RowInfo), 256) * 256;
    s.total = s.info_bytes + 8 * (long long)G.kv_heads * s.mean_rows * s.words;
    return s;
}

template <class T, int DP, int NG>
static void launch_bwd(const Geometry &G, const void *q, const void *k, const void *v, const int *idx, const void *out, const float *lse,
                       const void *dout, void *dq, void *dk, void *dv, char *ws, const BwdSpace &sp, hipStream_t st)
{
    RowInfo *info = (RowInfo *)ws;
    unsigned long long *bits = (unsigned long long *)(ws + sp.info_bytes);
    const int slices = (int)ceil_div(G.group, 16);
    const bool full = G.head_dim == DP;
    if (G.q_rows > 0) {
        const int per_tile = G.group < 16 ? 16 / G.group : 1;
#define NSP_GO(NT, WIDE)                                                                                                                     \
    hipLaunchKernelGGL((k_attend_dq<T, DP, NT, NG, WIDE>), dim3((unsigned)(ceil_div(G.q_rows, 4 * NT * per_tile) * slices * G.kv_heads)), \
                       dim3(256), 0, st, G, (const T *)q, (const T *)k, (const T *)v, idx, (const T *)out, lse, (const T *)dout, (T *)dq,    \
                       info, slices, per_tile)
        bool two = false;
        if constexpr (sizeof(T) == 2 && DP <= 128) {
            two = per_tile <= 8 && (long long)G.q_rows * slices * G.kv_heads >= 2 * per_tile * 2048LL;
            if (two) {
                if (G.block >= 16 * NG) NSP_GO(2, true); else NSP_GO(2, false);
            }
        }
        if (!two) {
            if (G.block >= 16 * NG) NSP_GO(1, true); else NSP_GO(1, false);
        }
#undef NSP_GO
        if (sp.mean_rows > 0)
            hipLaunchKernelGGL(k_pattern_bits, dim3((unsigned)((long long)sp.words * G.kv_heads)), dim3(256), 0, st, G, idx, bits,
                               sp.mean_rows, sp.words);
    }
    if (sp.mean_rows > 0) {
        const int parts = G.block > 64 ? G.block / 64 : 1;
        const dim3 grid((unsigned)(sp.mean_rows * G.kv_heads * parts)), block(G.block > 64 ? 256 : 4 * G.block);
        if (full)
            hipLaunchKernelGGL((k_attend_dkv<T, DP, true>), grid, block, 0, st, G, (const T *)q, (const T *)k, (const T *)v,
                               (const T *)dout, info, bits, (T *)dk, (T *)dv, sp.mean_rows, sp.words, parts);
        else
            hipLaunchKernelGGL((k_attend_dkv<T, DP, false>), grid, block, 0, st, G, (const T *)q, (const T *)k, (const T *)v,
                               (const T *)dout, info, bits, (T *)dk, (T *)dv, sp.mean_rows, sp.words, parts);
    }
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

int nsparse_lm_block_attention_bwd(const nsparse_lm_attn *a, const void *q, const void *k, const void *v, const int *idx, const void *out,
                                   const float *lse, const void *dout, void *dq, void *dk, void *dv, void *workspace,
                                   long long workspace_bytes, void *stream)
{
    using namespace nsp::lm;
    clear_error();
    Geometry G;
    if (int rc = geometry(a, true, true, &G)) return rc;
    if (G.page_size > 0) return fail(NSPARSE_LM_EARG, "block_attention_bwd: not for paged caches");
    const BwdSpace sp = bwd_space(G);
    if (sp.mean_rows * G.kv_heads > 0x7fffffffLL / 4) return fail(NSPARSE_LM_EARG, "block_attention_bwd: blocks x heads out of range");
    if ((G.q_rows > 0 && (!q || !idx || !out || !lse || !dout || !dq)) || (G.k_rows > 0 && (!k || !v || !dk || !dv)))
        return fail(NSPARSE_LM_EARG, "block_attention_bwd: a required pointer is NULL");
    if (((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)out | (uintptr_t)dout | (uintptr_t)dq | (uintptr_t)dk | (uintptr_t)dv |
         (uintptr_t)workspace) & 15)
        return fail(NSPARSE_LM_EALIGN, "block_attention_bwd: tensors and workspace begin at multiples of 16 bytes");
    if (sp.total > 0 && (!workspace || workspace_bytes < sp.total))
        return fail(NSPARSE_LM_EWORKSPACE, "block_attention_bwd: workspace smaller than nsparse_lm_block_attention_bwd_workspace() says");
    hipStream_t st = (hipStream_t)stream;
    char *ws = (char *)workspace;
#define NSP_DIM(T, NG)                                                                                                  \
    if (G.head_dim <= 64) launch_bwd<T, 64, NG>(G, q, k, v, idx, out, lse, dout, dq, dk, dv, ws, sp, st);               \
    else if (G.head_dim <= 128) launch_bwd<T, 128, NG>(G, q, k, v, idx, out, lse, dout, dq, dk, dv, ws, sp, st);        \
    else launch_bwd<T, 256, 2>(G, q, k, v, idx, out, lse, dout, dq, dk, dv, ws, sp, st)
    if (a->dtype == NSPARSE_LM_BF16) { NSP_DIM(__bf16, 4); }
    else if (a->dtype == NSPARSE_LM_F16) { NSP_DIM(_Float16, 4); }
    else { NSP_DIM(float, 2); }
#undef NSP_DIM
    return launched("block_attention_bwd");
}
}
