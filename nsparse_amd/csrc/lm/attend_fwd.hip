// attend_fwd.hip -- attention over the listed blocks of keys.
//
//   out[t,h] = sum_j p_j v_j,  p = softmax(scale q.k_j) over the keys j of the blocks that row (t, g) lists, g = h / group.
//
// One wavefront takes one pattern row: the group's query heads are the (up to 16) columns of its matrix products, so K and V are
// read once for all of them.  Nothing but registers: S^T = K Q^T comes out with lane l holding column (query) l % 16 and keys
// 4 (l / 16) + i, which, rounded, is already the right operand of O^T = V^T P^T; V is read row by row, E = DP / 16
// neighbouring columns a lane, and transposed inside the lane (common.h).  The softmax runs over the blocks with
// a running maximum and sum in 32 bits, in base 2.
// The probabilities are rounded to the inputs' type for the second product, half a step each, because products of 32-bit operands run at a
// seventh of the rate (152 against 1107 TFLOP/s); their sum is taken before that.  That error is about as large as the output's own rounding: against 64 bits the outputs
// are off by 1.1 to 1.4 times (rms) what the rounding of exact outputs alone would leave.  Single precision rounds nothing.
// Prompts: a workgroup takes several neighbouring rows, 4 NT x (16 / heads of the group) of them, as the columns of the products of its
// four wavefronts, and walks the union of their blocks (attend.h): a block that neighbours share is read from the L2 cache
// once, into LDS.  The next block is asked for before this one's products, but the compiler cannot tell the halves of kt and vt apart and waits
// for it before the first read of LDS: what hides the way to memory is the other workgroup of the compute unit.
// With few rows (a serving step) eight wavefronts share a row: wavefront w takes every eighth tile of keys and the partial
// results meet in LDS.
// Measured, 32 query and 8 key heads of 128, 16 blocks of 64, bf16.  8192 rows of a prompt whose neighbours agree on part of their blocks: 402 us, 311 TFLOP/s
// over the listed keys; bound by that wait, by LDS (a wavefront reads as many cycles of operands as its products take) and by blocks that only
// some of the workgroup's rows list.  64 conversations, one row each, 32 blocks: 46 us, 4.2 TB/s, bound by memory.  One row: 15 us, bound by latency.
#include "attend.h"

namespace nsp {
namespace lm {

template <class T, int DP, int NG, bool FULL, int WAVES>
__global__ void __launch_bounds__(WAVES > 1 ? 64 * WAVES : 256)
    k_attend(const Geometry G, const T *__restrict__ q, const T *__restrict__ k, const T *__restrict__ v, const int *__restrict__ idx,
             T *__restrict__ out, float *__restrict__ lse, int slices)
{
    constexpr int KS = DP / 32, E = DP / 16;
    const int lane = lane_id(), col = lane & 15, quad = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    // consecutive workgroups go round the key heads: with 8 of them each XCD's cache serves one head's keys
    const int g = (int)(group_id() % G.kv_heads);
    const int rest = (int)(group_id() / G.kv_heads);
    const int slice = rest % slices;
    const int t = WAVES > 1 ? rest / slices : (rest / slices) * 4 + wave;
    if (t >= G.q_rows) return;
    Seq sq;
    const int i = seq_of_query(G, t, sq);
    if (i < 0) return;  // the same for every wavefront that shares a row
    const int limit = visible_keys(G, sq, i);
    const int D = G.head_dim;
    const int h0 = g * G.group + slice * 16;
    const int nh = G.group - slice * 16 < 16 ? G.group - slice * 16 : 16;

    Frag<T> qf[KS];
    row_frags<T, KS, FULL>(qf, q + (long long)t * G.q_row + (long long)(h0 + col) * G.q_head, quad, D, col < nh);
    const float sl2 = G.scale * kLog2e;
    f32x4 o[E];
#pragma unroll
    for (int j = 0; j < E; j++) o[j] = f32x4{0, 0, 0, 0};
    float m = -INFINITY, l = 0.f;
    const int shift = 27 - __builtin_clz(G.block);  // log2(block / 16)
    const int *row = idx + ((long long)t * G.kv_heads + g) * G.width;
    int seen = -1;
    for (int at = 0; at < G.width && limit > 0; at += 64) {
        const Chunk c = chunk_of_row(G, sq, g, row, at, limit, seen);
        const int total = c.n << shift;
        for (int u = (WAVES > 1 ? wave : 0) * NG; u < total; u += NG * WAVES) {
            Group16 x[NG];
            bool whole = true;
#pragma unroll
            for (int y = 0; y < NG; y++) {
                x[y] = group_of_chunk(G, c, u + y, shift, g);
                whole = whole && x[y].rows == 16;
            }
            // with few rows nobody else hides the way to memory: everything is asked for at once
            constexpr bool kEarly = WAVES > 1;
            Rows<T, E> ve[kEarly ? NG / 2 : 1];
            auto load_v = [&](Rows<T, E> &vr, int y) {
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const Group16 &gx = x[y + (e >> 2)];
                    const int r = 4 * quad + (e & 3);
                    const T *p = v + gx.v_off + (long long)(r < gx.rows ? r : 0) * G.v_row + col * E;
                    if constexpr (FULL) rows_load(vr, e, p); else rows_load_part(vr, e, p, D - col * E);
                }
            };
            // S^T, sixteen keys at a time
            f32x4 s[NG];
            if constexpr (kEarly) {
                Frag<T> kf[NG][KS];
#pragma unroll
                for (int y = 0; y < NG; y++)
                    row_frags<T, KS, FULL>(kf[y], k + x[y].k_off + (long long)(col < x[y].rows ? col : 0) * G.k_row, quad, D, true);
#pragma unroll
                for (int y = 0; y < NG; y += 2) load_v(ve[y / 2], y);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int y = 0; y < NG; y++) {
                    s[y] = f32x4{0, 0, 0, 0};
#pragma unroll
                    for (int z = 0; z < KS; z++) s[y] = mma(kf[y][z], qf[z], s[y]);
                }
            } else {
#pragma unroll
                for (int y = 0; y < NG; y++) {
                    Frag<T> kf[KS];
                    row_frags<T, KS, FULL>(kf, k + x[y].k_off + (long long)(col < x[y].rows ? col : 0) * G.k_row, quad, D, true);
                    s[y] = f32x4{0, 0, 0, 0};
#pragma unroll
                    for (int z = 0; z < KS; z++) s[y] = mma(kf[z], qf[z], s[y]);
                }
            }
            float top = -INFINITY;
#pragma unroll
            for (int y = 0; y < NG; y++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    s[y][e] = 4 * quad + e < x[y].rows ? s[y][e] * sl2 : -INFINITY;
                    top = fmaxf(top, s[y][e]);
                }
            top = quads_max(top);
            const float m_new = fmaxf(m, top);
            const float m_use = m_new == -INFINITY ? 0.f : m_new;
            if (__any(m_new > m)) {
                const float alpha = pow2(m - m_use);  // 0 while m is -inf
                l *= alpha;
#pragma unroll
                for (int j = 0; j < E; j++) o[j] *= alpha;
                m = m_new;
            }
#pragma unroll
            for (int y = 0; y < NG; y++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    s[y][e] = pow2(s[y][e] - m_use);
                    l += s[y][e];
                }
            // O^T += V^T P^T, 32 keys at a time
#pragma unroll
            for (int y = 0; y < NG; y += 2) {
                Rows<T, E> late;
                if constexpr (!kEarly) load_v(late, y);
                Rows<T, E> &vr = kEarly ? ve[y / 2] : late;
                // a hidden key's row must not reach the sum, whatever stands there
                if (!whole) {
#pragma unroll
                    for (int e = 0; e < 8; e++)
                        if (4 * quad + (e & 3) >= x[y + (e >> 2)].rows) rows_clear(vr, e);
                }
                const Frag<T> pf = frag_pack<T>(s[y], s[y + 1]);
#pragma unroll
                for (int j = 0; j < E; j++) o[j] = mma(rows_column(vr, j), pf, o[j]);
            }
        }
    }
    l = quads_sum(l);
    T *orow = out + ((long long)t * G.heads + h0 + col) * D;
    if constexpr (WAVES == 1) {
        if (col < nh) {
            const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                float w[E];
#pragma unroll
                for (int j = 0; j < E; j++) w[j] = o[j][e] * inv;
                const int d = (4 * quad + e) * E;
                store_columns<T, E>(orow + d, w, D - d);
            }
            if (lse && quad == 0) lse[(long long)t * G.heads + h0 + col] = l == 0.f ? -INFINITY : (m + log2f(l)) * kLn2;
        }
    } else {
        constexpr int LD = DP + 4;
        __shared__ float part[WAVES * 16 * LD];
        __shared__ float ml[2 * WAVES * 16];
        if (quad == 0) {
            ml[wave * 16 + col] = m;
            ml[(WAVES + wave) * 16 + col] = l;
        }
        __syncthreads();
        float M = -INFINITY;
#pragma unroll
        for (int w = 0; w < WAVES; w++) M = fmaxf(M, ml[w * 16 + col]);
        const float M_use = M == -INFINITY ? 0.f : M;
        float L = 0.f;
#pragma unroll
        for (int w = 0; w < WAVES; w++) L += ml[(WAVES + w) * 16 + col] * pow2(ml[w * 16 + col] - M_use);
        const float mine = (L == 0.f ? 0.f : 1.f / L) * pow2(m - M_use);
#pragma unroll
        for (int e = 0; e < 4; e++)
#pragma unroll
            for (int j = 0; j < E; j++) part[(wave * 16 + col) * LD + (4 * quad + e) * E + j] = o[j][e] * mine;
        if (lse && wave == 0 && quad == 0 && col < nh)
            lse[(long long)t * G.heads + h0 + col] = L == 0.f ? -INFINITY : (M + log2f(L)) * kLn2;
        __syncthreads();
        for (int x = threadIdx.x; x < nh * DP; x += 64 * WAVES) {
            const int hh = x / DP, d = x % DP;
            if (!FULL && d >= D) continue;
            float a = 0.f;
#pragma unroll
            for (int w = 0; w < WAVES; w++) a += part[(w * 16 + hh) * LD + d];
            out[((long long)t * G.heads + h0 + hh) * D + d] = from_f32<T>(a);
        }
    }
}

// ---- prompts ---------------------------------------------------------------------------------------------------------------
template <class T, int DP, int NT, int NG, bool WIDE>
__global__ void __launch_bounds__(256, DP * sizeof(T) <= 256 ? 2 : 1)
    k_attend_tiles(const Geometry G, const T *__restrict__ q, const T *__restrict__ k, const T *__restrict__ v, const int *__restrict__ idx,
                   T *__restrict__ out, float *__restrict__ lse, int slices, int per_tile)
{
    constexpr int KS = DP / 32, E = DP / 16, kTile = NG * 16 * Tile<T, DP>::kPieces;
    __shared__ u32x4 kt[2][kTile], vt[2][kTile];
    __shared__ Union un;
    const int wave = uniform((int)(threadIdx.x >> 6));
    // consecutive workgroups go round the key heads: with 8 of them each XCD's cache serves one head's keys
    const int g = (int)(group_id() % G.kv_heads);
    const int rest = (int)(group_id() / G.kv_heads);
    const int slice = rest % slices;
    const int per_wave = NT * per_tile;  // rows a wavefront
    const int t0 = (rest / slices) * 4 * per_wave;
    const int t1 = t0 + 4 * per_wave < G.q_rows ? t0 + 4 * per_wave : G.q_rows;
    const int D = G.head_dim;
    const float sl2 = fmaxf(fabsf(G.scale) * kLog2e, 1e-37f);  // a negative scale's sign goes to q; 0 x -inf is no score

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
        // lane i's row for the walk; a column's row is number (wave * NT + x) * per_tile + Column::sub
        const int t_mine = t0 + opaque(lane_id());
        const int limit = t_mine >= a && t_mine < z ? visible_keys(G, sq, (int)(t_mine - sq.q_base)) : 0;
        Frag<T> qf[NT][KS];
        int lim[NT], num[NT];
#pragma unroll
        for (int x = 0; x < NT; x++) {
            num[x] = (wave * NT + x) * per_tile + c0.sub;
            const bool on = c0.live && t0 + num[x] >= a && t0 + num[x] < z;
            lim[x] = pull(limit, num[x]);
            if (!on) lim[x] = 0;
            row_frags<T, KS, false>(qf[x], q + (long long)(on ? t0 + num[x] : a) * G.q_row + (long long)c0.head * G.q_head, quad, D, on);
            if (G.scale < 0) {
#pragma unroll
                for (int w = 0; w < KS; w++) frag_negate(qf[x][w]);
            }
        }
        const int count = z - a;
        const unsigned long long every = (count < 64 ? (1ULL << count) - 1 : ~0ULL) << (a - t0);
        unsigned long long todo = every, now = every;
        while (todo) {
            f32x4 o[NT][E];
            float m[NT], l[NT];
#pragma unroll
            for (int x = 0; x < NT; x++) {
                m[x] = -INFINITY;
                l[x] = 0.f;
#pragma unroll
                for (int j = 0; j < E; j++) o[x][j] = f32x4{0, 0, 0, 0};
            }
            const int blocks = (read_lane(limit, 63 - __builtin_clzll(now)) + G.block - 1) / G.block;
            for (int b0 = 0; b0 < blocks; b0 += kRange) {
                union_build(un, G, idx, g, t0, now, limit, b0, blocks - b0 < kRange ? blocks - b0 : kRange, wave);
                const int steps = walk_steps<NG, WIDE>(G, un);
                if (steps == 0) continue;
                Step<NG, WIDE> st;
                walk_step<NG, WIDE>(st, G, sq, g, un, b0, limit, 0);
                tile_load<T, DP, NG, WIDE>(kt[0], k, st.k_off, st, G.k_row, D);
                tile_load<T, DP, NG, WIDE>(vt[0], v, st.v_off, st, G.v_row, D);
                __syncthreads();
                for (int step = 0; step < steps; step++) {
                    const int buf = step & 1;
                    const bool more = step + 1 < steps;
                    Step<NG, WIDE> next = st;
                    if (more) {
                        walk_step<NG, WIDE>(next, G, sq, g, un, b0, limit, step + 1);
                        tile_load<T, DP, NG, WIDE>(kt[buf ^ 1], k, next.k_off, next, G.k_row, D);
                        tile_load<T, DP, NG, WIDE>(vt[buf ^ 1], v, next.v_off, next, G.v_row, D);
                    }
                    const bool use = (st.any >> (wave * NT * per_tile)) & (NT * per_tile < 64 ? (1ULL << (NT * per_tile)) - 1 : ~0ULL);
                    Frag<T> pf[NT][NG / 2];
                    if (use) {
                        f32x4 s[NT][NG];
#pragma unroll
                        for (int y = 0; y < NG; y++)
#pragma unroll
                            for (int x = 0; x < NT; x++) s[x][y] = f32x4{0, 0, 0, 0};
                        pipelined<Frag<T>, NG * KS, 4, 2>(
                            [&](int i) { return tile_frag<T, DP>(kt[buf], 16 * (i / KS) + col, i % KS, quad); },
                            [&](int i, const Frag<T> &f) {
#pragma unroll
                                for (int x = 0; x < NT; x++) s[x][i / KS] = mma(f, qf[x][i % KS], s[x][i / KS]);
                            });
#pragma unroll
                        for (int x = 0; x < NT; x++) {
                            if (NT > 1 && !((st.any >> ((wave * NT + x) * per_tile)) & ((1ULL << per_tile) - 1))) {
#pragma unroll
                                for (int y = 0; y < NG; y += 2) pf[x][y / 2] = frag_zero<T>();
                                continue;
                            }
                            bool on[NG];
                            bool all = WIDE;
#pragma unroll
                            for (int y = 0; y < NG; y++) on[y] = (st.lists(y) >> num[x]) & 1;
                            if (WIDE) all = __all(!on[0] || lim[x] - st.from[0] >= 16 * NG);
                            if (!all) {
                                // some column does not see every key of a block that it lists
#pragma unroll
                                for (int y = 0; y < NG; y++) {
                                    const int vis = on[y] ? lim[x] - st.first(y) - 4 * quad : 0;
#pragma unroll
                                    for (int e = 0; e < 4; e++) s[x][y][e] = e < vis ? s[x][y][e] : -INFINITY;
                                }
                            }
                            float top = -INFINITY;
#pragma unroll
                            for (int y = 0; y < NG; y++)
#pragma unroll
                                for (int e = 0; e < 4; e++) top = fmaxf(top, s[x][y][e]);
                            top = quads_max(top) * sl2;
                            if (WIDE && !on[0]) top = -INFINITY;
                            // the maximum need not be the true one: sums of powers up to 2^8 are as exact
                            if (__any(top > m[x] + 8.f)) {
                                const float m_new = fmaxf(m[x], top);
                                const float alpha = pow2(m[x] - (m_new == -INFINITY ? 0.f : m_new));
                                l[x] *= alpha;
#pragma unroll
                                for (int j = 0; j < E; j++) o[x][j] *= alpha;
                                m[x] = m_new;
                            }
                            // columns that do not list the block: 2^-inf
                            const float base = (WIDE && !on[0]) ? INFINITY : m[x] == -INFINITY ? 0.f : m[x];
#pragma unroll
                            for (int y = 0; y < NG; y++)
#pragma unroll
                                for (int e = 0; e < 4; e++) {
                                    s[x][y][e] = pow2(__builtin_fmaf(s[x][y][e], sl2, -base));
                                    l[x] += s[x][y][e];
                                }
#pragma unroll
                            for (int y = 0; y < NG; y += 2) pf[x][y / 2] = frag_pack<T>(s[x][y], s[x][y + 1]);
                        }
                    }
                    if (use) {
                        if constexpr (sizeof(T) == 2) {
                            pipelined<Frag<T>, NG / 2 * E, 4, 2>(
                                [&](int i) { return Columns<T, DP>(vt[buf], 2 * (i / E), quad, col).frag(i % E); },
                                [&](int i, const Frag<T> &f) {
#pragma unroll
                                    for (int x = 0; x < NT; x++) o[x][i % E] = mma(f, pf[x][i / E], o[x][i % E]);
                                });
                        } else {
#pragma unroll
                            for (int y = 0; y < NG; y += 2) {
                                const Columns<T, DP> c(vt[buf], y, quad, col);
#pragma unroll
                                for (int j = 0; j < E; j++) {
                                    const Frag<T> f = c.frag(j);
#pragma unroll
                                    for (int x = 0; x < NT; x++) o[x][j] = mma(f, pf[x][y / 2], o[x][j]);
                                }
                            }
                        }
                    }
                    st = next;
                    __syncthreads();
                }
            }
            // A value that is no number reaches the columns that do not see it as 0 x NaN: then every row by itself, whose hidden keys are
            // zeros in LDS.
            bool bad = false;
#pragma unroll
            for (int x = 0; x < NT; x++) {
                l[x] = quads_sum(l[x]);
                float t = l[x];
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
                const int n = (wave * NT + x) * per_tile + c1.sub;
                if (!c1.live || !((now >> n) & 1)) continue;
                const long long th = (long long)(t0 + n) * G.heads + c1.head;
                store_row<T, DP>(out + th * D, o[x], l[x] == 0.f ? 0.f : 1.f / l[x], c1.quad, D);
                if (lse && c1.quad == 0) lse[th] = l[x] == 0.f ? -INFINITY : (m[x] + log2f(l[x])) * kLn2;
            }
            todo &= ~now;
            now = todo & -todo;
        }
        a = z;
    }
}

template <class T, int DP, int NT, int NG>
static void launch_tiles(const Geometry &G, const void *q, const void *k, const void *v, const int *idx, void *out, float *lse, hipStream_t st)
{
    const int slices = (int)ceil_div(G.group, 16);
    const int per_tile = G.group < 16 ? 16 / G.group : 1;
    const dim3 grid = groups(ceil_div(G.q_rows, 4 * NT * per_tile) * slices * G.kv_heads);
    if (NG == 4 || G.block >= 16 * NG)
        launch((k_attend_tiles<T, DP, NT, NG, true>), grid, dim3(256), 0, st, G, (const T *)q, (const T *)k, (const T *)v, idx,
                           (T *)out, lse, slices, per_tile);
    else if constexpr (NG == 2)
        launch((k_attend_tiles<T, DP, NT, NG, false>), grid, dim3(256), 0, st, G, (const T *)q, (const T *)k, (const T *)v, idx,
                           (T *)out, lse, slices, per_tile);
}

template <class T, int DP, int NG>
static void launch_attend(const Geometry &G, const void *q, const void *k, const void *v, const int *idx, void *out, float *lse, hipStream_t st)
{
    const int slices = (int)ceil_div(G.group, 16);
    const long long rows = (long long)G.q_rows * slices;
    // several wavefronts a row while that leaves compute units without work otherwise (8 key heads, 16 blocks of 64: 64 sequences 47
    // against 83 us, 128: 107 and 108; 4 key heads, 8 blocks of 32: 512 sequences 31.5 against 25.6)
    const bool split = rows * G.kv_heads < 2048;
    const bool full = G.head_dim == DP;
    // neighbouring rows together where there are some (256 sequences of 3 new tokens: 357 against 297 us row by row, of 4: 224;
    // but 512 of 2, 2 heads each and blocks of 16: 57 against 200)
    if (!split && G.q_rows / G.n_seq >= 4) {
        // 64 keys a step where a block has them, else 32 (blocks of 32 in steps of 64: 55 against 39 us for 3945 rows of 16 heads)
        const int per_tile = G.group < 16 ? 16 / G.group : 1;
        if constexpr (sizeof(T) == 2 && DP <= 128) {
            if (G.block >= 64) {
                // two sets of columns read half as much of LDS a product, but neighbours have to agree on more blocks (8192 rows, 32/8 heads: 442 against
                // 549 us with one set where few agree, 305 against 274 where sixteen rows agree on all but one; 2048 rows, 64/4 heads: 92 against 111)
                if (per_tile <= 8 && rows * G.kv_heads >= 2 * per_tile * 2048LL) launch_tiles<T, DP, 2, 4>(G, q, k, v, idx, out, lse, st);
                else launch_tiles<T, DP, 1, 4>(G, q, k, v, idx, out, lse, st);
                return;
            }
        }
        launch_tiles<T, DP, 1, 2>(G, q, k, v, idx, out, lse, st);
        return;
    }
#define NSP_GO(FULL, WAVES)                                                                                                          \
    launch((k_attend<T, DP, NG, FULL, WAVES>), groups((WAVES > 1 ? rows : ceil_div(G.q_rows, 4) * slices) * G.kv_heads), \
                       dim3(WAVES > 1 ? 64 * WAVES : 256), 0, st, G, (const T *)q, (const T *)k, (const T *)v, idx, (T *)out, lse, slices)
    if (split) {
        constexpr int kSplit = DP * sizeof(T) > 512 ? 4 : 8;  // registers for a row's sums and a step's keys and values
        if (full) NSP_GO(true, kSplit); else NSP_GO(false, kSplit);
    } else {
        if (full) NSP_GO(true, 1); else NSP_GO(false, 1);
    }
#undef NSP_GO
}

}  // namespace lm
}  // namespace nsp

extern "C" int nsparse_lm_block_attention(const nsparse_lm_attn *a, const void *q, const void *k, const void *v, const int *idx, void *out,
                                          float *lse, void *stream)
{
    using namespace nsp::lm;
    clear_error();
    Geometry G;
    if (int rc = geometry(a, true, true, &G)) return rc;
    if (G.q_rows == 0) return 0;
    if (!q || !idx || !out || (G.k_rows > 0 && (!k || !v))) return fail(NSPARSE_LM_EARG, "block_attention: a required pointer is NULL");
    if (((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)out) & 15)
        return fail(NSPARSE_LM_EALIGN, "block_attention: q, k, v and out begin at multiples of 16 bytes");
    hipStream_t st = (hipStream_t)stream;
#define NSP_DIM(T, NG)                                                              \
    if (G.head_dim <= 64) launch_attend<T, 64, NG>(G, q, k, v, idx, out, lse, st);  \
    else if (G.head_dim <= 128) launch_attend<T, 128, NG>(G, q, k, v, idx, out, lse, st); \
    else launch_attend<T, 256, 2>(G, q, k, v, idx, out, lse, st)
    if (a->dtype == NSPARSE_LM_BF16) { NSP_DIM(__bf16, 4); }
    else if (a->dtype == NSPARSE_LM_F16) { NSP_DIM(_Float16, 4); }
    else { NSP_DIM(float, 2); }
#undef NSP_DIM
    return launched("block_attention");
}
