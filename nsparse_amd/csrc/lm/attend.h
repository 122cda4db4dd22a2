// attend.h -- keys of the selected blocks, sixteen at a time, as the attention kernels walk them.
#pragma once
#include "common.h"

namespace nsp {
namespace lm {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

// The (up to 64) blocks of a pattern chunk, one per lane: where the block's keys begin (elements from k and v, the head's
// offset included) and how many of them the query sees.
struct Chunk {
    long long k_off, v_off;
    int rows;
    int n;  // blocks (uniform)
};

__device__ inline Chunk chunk_of_row(const Geometry &G, const Seq &sq, int g, const int *row, int at, int limit, int &seen)
{
    Chunk c;
    int b;
    c.n = pattern_chunk(row, at, G.width, (limit + G.block - 1) / G.block, seen, b);
    const bool mine = lane_id() < c.n;
    c.k_off = (long long)g * G.k_head;
    c.v_off = (long long)g * G.v_head;
    c.rows = 0;
    if (mine) {
        const int left = limit - b * G.block;
        if (G.page_size > 0) {
            const long long page = page_of_block(G, sq.s, b);
            if (page >= 0) {
                const long long in = (long long)(b % G.per_page) * G.block;
                c.k_off += page * G.k_page + in * G.k_row;
                c.v_off += page * G.v_page + in * G.v_row;
                c.rows = left < G.block ? left : G.block;
            }
        } else {
            const long long r = sq.k_base + (long long)b * G.block;
            c.k_off += r * G.k_row;
            c.v_off += r * G.v_row;
            c.rows = left < G.block ? left : G.block;
        }
    }
    return c;
}

// Group u (sixteen keys) of a chunk: offsets and visible keys; a group behind the last one has none and points at the
// head's first key, which exists.
struct Group16 {
    long long k_off, v_off;
    int rows;
};
__device__ inline Group16 group_of_chunk(const Geometry &G, const Chunk &c, int u, int shift, int g)
{
    Group16 x{(long long)g * G.k_head, (long long)g * G.v_head, 0};
    const int e = u >> shift;
    if (e < c.n) {
        const int sub = (u & ((1 << shift) - 1)) << 4;
        const int left = read_lane(c.rows, e) - sub;
        if (left > 0) {
            x.k_off = read_lane64(c.k_off, e) + (long long)sub * G.k_row;
            x.v_off = read_lane64(c.v_off, e) + (long long)sub * G.v_row;
            x.rows = left < 16 ? left : 16;
        }
    }
    return x;
}

// keys a query of position len_k - len_q + i sees
__device__ inline int visible_keys(const Geometry &G, const Seq &sq, int i)
{
    if (!G.causal) return sq.k_len;
    const int lim = sq.k_len - sq.q_len + i + 1;
    return lim < 0 ? 0 : lim;
}

// ---- several query rows at once -------------------------------------------------------------------------------------------
// The rows of neighbouring queries list mostly the same blocks.  A workgroup that has up to 64 of them walks the union of their
// rows: for a range of blocks, one word a block says which queries list it, and the blocks with a word that is not 0, upwards,
// are the walk.
constexpr int kRange = 1024;
struct Union {
    unsigned long long who[kRange];
    unsigned short list[kRange];
    int n;
};
// By a workgroup of four wavefronts: blocks b0 .. b0 + nb of the rows t0 + i, i in `now`; lane i holds row i's visible keys.
__device__ inline void union_build(Union &u, const Geometry &G, const int *idx, int g, int t0, unsigned long long now, int limit, int b0, int nb,
                                   int wave)
{
    const int lane = opaque(lane_id());
    __syncthreads();
    for (int x = wave * 64 + lane; x < nb; x += 256) u.who[x] = 0;
    __syncthreads();
    if (G.width <= 16) {
        // four rows at a time, sixteen lanes each; all of them are on their way before the first is looked at
        const int sub = lane >> 4, j = lane & 15;
        int e[4];
#pragma unroll
        for (int p = 0; p < 4; p++) {
            const int n = 16 * p + 4 * wave + sub;
            e[p] = ((now >> n) & 1) && j < G.width ? idx[((long long)(t0 + n) * G.kv_heads + g) * G.width + j] : -1;
        }
#pragma unroll
        for (int p = 0; p < 4; p++) {
            const int n = 16 * p + 4 * wave + sub;
            if (!((now >> (16 * p + 4 * wave)) & 15)) continue;
            int top = e[p], o;  // greatest entry up to and including this lane's
            o = __builtin_amdgcn_update_dpp(-1, top, 0x111, 0xf, 0xf, false);
            top = o > top ? o : top;
            o = __builtin_amdgcn_update_dpp(-1, top, 0x112, 0xf, 0xf, false);
            top = o > top ? o : top;
            o = __builtin_amdgcn_update_dpp(-1, top, 0x114, 0xf, 0xf, false);
            top = o > top ? o : top;
            o = __builtin_amdgcn_update_dpp(-1, top, 0x118, 0xf, 0xf, false);
            top = o > top ? o : top;
            const int before = __builtin_amdgcn_update_dpp(-1, top, 0x111, 0xf, 0xf, false);
            const int lim = pull(limit, n), b = e[p];
            if (b > before && (long long)b * G.block < lim && b >= b0 && b < b0 + nb) atomicOr((unsigned *)&u.who[b - b0] + (n >> 5), 1u << (n & 31));
        }
    } else {
        for (int n = wave; n < 64; n += 4) {
            if (!((now >> n) & 1)) continue;
            const int lim = read_lane(limit, n);
            const int *row = idx + ((long long)(t0 + n) * G.kv_heads + g) * G.width;
            int seen = -1;
            for (int at = 0; at < G.width; at += 64) {
                int b;
                const int c = pattern_chunk(row, at, G.width, (lim + G.block - 1) / G.block, seen, b);
                if (lane < c && b >= b0 && b < b0 + nb) atomicOr((unsigned *)&u.who[b - b0] + (n >> 5), 1u << (n & 31));
            }
        }
    }
    __syncthreads();
    if (wave == 0) {
        int n = 0;
        for (int x = 0; x < nb; x += 64) {
            const bool in = x + lane < nb && u.who[x + lane] != 0;
            const unsigned long long m = __ballot(in);
            if (in) u.list[n + __popcll(m & ((1ULL << lane) - 1))] = (unsigned short)(x + lane);
            n += __popcll(m);
        }
        if (lane == 0) u.n = n;
    }
    __syncthreads();
}

// What a column of a wavefront's products stands for: the tile's row `sub` and a query head.  Asked for where it is needed.
struct Column {
    int col, quad, sub, head;
    bool live;
    __device__ inline Column(const Geometry &G, int g, int slice, int per_tile)
    {
        const int lane = opaque(lane_id());
        col = lane & 15;
        quad = lane >> 4;
        const int heads = G.group < 16 ? G.group : 16;  // columns a row
        sub = col / heads;
        live = sub < per_tile && slice * 16 + col % heads < G.group;
        head = g * G.group + slice * 16 + (live ? col % heads : 0);
        if (sub >= per_tile) sub = 0;
    }
};

// NG groups of sixteen keys of a walk.  WIDE: a block has at least as many, they are neighbours; else up to NG blocks.
template <int NG, bool WIDE> struct Step {
    static constexpr int kParts = WIDE ? 1 : NG;
    long long k_off[kParts], v_off[kParts];  // elements from k and v, the head's offset included
    int from[kParts], left[kParts];          // first key inside the sequence; keys from there on that some listing query sees
    unsigned long long who[kParts], any;     // queries that list the block
    __device__ inline int first(int y) const { return WIDE ? from[0] + 16 * y : from[y]; }
    __device__ inline unsigned long long lists(int y) const { return who[WIDE ? 0 : y]; }
};
template <int NG, bool WIDE> __device__ inline int walk_steps(const Geometry &G, const Union &u)
{
    const int groups = uniform(u.n) * (G.block >> 4);
    return (groups + NG - 1) / NG;
}
template <int NG, bool WIDE>
__device__ inline void walk_step(Step<NG, WIDE> &s, const Geometry &G, const Seq &sq, int g, const Union &u, int b0, int limit, int step)
{
    const int shift = 27 - __builtin_clz(G.block), groups = uniform(u.n) << shift;
    s.any = 0;
#pragma unroll
    for (int y = 0; y < Step<NG, WIDE>::kParts; y++) {
        const int i = step * NG + y;
        s.k_off[y] = (long long)g * G.k_head;
        s.v_off[y] = (long long)g * G.v_head;
        s.from[y] = 0;
        s.left[y] = 0;
        s.who[y] = 0;
        if (i >= groups) continue;
        const int e = uniform(u.list[i >> shift]), b = b0 + e;
        const unsigned long long who = uniform64(u.who[e]);
        const int part = i & ((1 << shift) - 1);
        const int start = b * G.block + part * 16;
        // the last of the listing rows sees the most
        int left = read_lane(limit, 63 - __builtin_clzll(who)) - start;
        const int end = (WIDE ? NG * 16 : 16);
        long long r = sq.k_base + start, page = 0;
        if (G.page_size > 0) {
            page = page_of_block(G, sq.s, b);
            if (page < 0) left = 0;
            r = (long long)(b % G.per_page) * G.block + part * 16;
        }
        if (left <= 0) continue;
        s.k_off[y] += page * G.k_page + r * G.k_row;
        s.v_off[y] += page * G.v_page + r * G.v_row;
        s.from[y] = start;
        s.left[y] = left < end ? left : end;
        s.who[y] = who;
        s.any |= who;
    }
}

// ---- keys and values in LDS ---------------------------------------------------------------------------------------------
// Rows of DP elements in pieces of 16 bytes; piece c of row r stands at c ^ (r % 16) (modulo the row), so that sixteen rows' equal
// pieces, which the fragments of a product read, lie in different banks, and a whole row, which the transposing read
// wants, stays in one stretch.  Columns behind head_dim and keys that nobody sees hold zeros.
template <class T, int DP> struct Tile {
    static constexpr int kPieces = DP * (int)sizeof(T) / 16;
    static constexpr int kSwizzle = kPieces < 16 ? kPieces - 1 : 15;
    static constexpr int kPer = 16 / (int)sizeof(T);  // elements a piece
    static __device__ inline int at(int r, int c) { return r * kPieces + (c ^ (r & kSwizzle)); }
};
template <class T, int DP> __device__ inline Frag<T> tile_frag(const u32x4 *t, int r, int s, int quad)
{
    if constexpr (sizeof(T) == 2) {
        return Frag<T>{t[Tile<T, DP>::at(r, 4 * s + quad)]};
    } else {
        const int c = 8 * s + 2 * quad;
        return Frag<T>{__builtin_bit_cast(f32x4, t[Tile<T, DP>::at(r, c)]), __builtin_bit_cast(f32x4, t[Tile<T, DP>::at(r, c + 1)])};
    }
}
// A transposed operand: slots 0 .. 3 are rows 4 quad + i of group y, slots 4 .. 7 those of group y + 1.  Sixteen-bit types: the
// LDS unit transposes 4 rows x 16 columns for sixteen lanes at a time, lane i of them names columns 4 (i % 4) of row i / 4 and gets
// column i of the four rows; row m of fragment j is column 16 j + m.  Single precision: E neighbouring columns a lane and row, row m of
// fragment j is column E m + j (as in rows_column).
typedef __attribute__((ext_vector_type(4))) short s16x4;
template <class T, int DP> struct Columns {
    const u32x4 *t;
    int y;
    __device__ inline Columns(const u32x4 *tile, int group, int quad, int col) : t(tile), y(group), q(quad), c(col) {}
    __device__ inline Frag<T> frag(int j) const
    {
        const int r = 16 * y + 4 * q + (c >> 2), piece = 2 * j + ((c & 3) >> 1);
        const u32x4 *p0 = t + Tile<T, DP>::at(r, piece), *p1 = t + Tile<T, DP>::at(r + 16, piece);
        typedef __attribute__((address_space(3))) s16x4 *lds;
        const u32x2 a = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds)((const u32x2 *)p0 + (c & 1))));
        const u32x2 b = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds)((const u32x2 *)p1 + (c & 1))));
        return Frag<T>{u32x4{a[0], a[1], b[0], b[1]}};
    }
    int q, c;
};
template <int DP> struct Columns<float, DP> {
    static constexpr int E = DP / 16;
    Rows<float, E> x;
    __device__ inline Columns(const u32x4 *t, int y, int quad, int col)
    {
#pragma unroll
        for (int s = 0; s < 8; s++)
#pragma unroll
            for (int c = 0; c < E / 4; c++) {
                const u32x4 v = t[Tile<float, DP>::at(16 * (y + (s >> 2)) + 4 * quad + (s & 3), col * (E / 4) + c)];
#pragma unroll
                for (int i = 0; i < 4; i++) x.w[s][4 * c + i] = __uint_as_float(v[i]);
            }
    }
    __device__ inline Frag<float> frag(int j) const { return rows_column(x, j); }
};
// o[j][e] * f of a product with Columns, to an output row
template <class T, int DP> __device__ inline void store_row(T *p, const f32x4 (&o)[DP / 16], float f, int quad, int head_dim)
{
    constexpr int E = DP / 16;
    if constexpr (sizeof(T) == 2) {
#pragma unroll
        for (int j = 0; j < E; j++) {
            const int d = 16 * j + 4 * quad;
            if (d < head_dim) *(u32x2 *)(p + d) = u32x2{pack2(o[j][0] * f, o[j][1] * f, T{}), pack2(o[j][2] * f, o[j][3] * f, T{})};
        }
    } else {
#pragma unroll
        for (int e = 0; e < 4; e++) {
            float w[E];
#pragma unroll
            for (int j = 0; j < E; j++) w[j] = o[j][e] * f;
            const int d = (4 * quad + e) * E;
            store_columns<T, E>(p + d, w, head_dim - d);
        }
    }
}
// 16 bytes a lane from memory to LDS without registers: lane i's land at the wavefront's `to` + 16 i.  They are there after the next barrier; the
// compiler waits for them earlier, before a read of the LDS array that they go to, whatever part of it is read.
// What is not there (behind head_dim, rows that nobody sees) comes from 16 bytes of zeros.
static __device__ const u32x4 kNothing[1] = {};
__device__ inline void fetch(u32x4 *to, const void *from, bool there)
{
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)(there ? from : kNothing),
                                     (__attribute__((address_space(3))) void *)to, 16, 0, 0);
}
// A step's keys (or values) to LDS, by 256 threads.
template <class T, int DP, int NG, bool WIDE>
__device__ inline void tile_load(u32x4 *t, const T *p, const long long (&off)[WIDE ? 1 : NG], const Step<NG, WIDE> &s, long long stride, int head_dim)
{
    constexpr int kPieces = Tile<T, DP>::kPieces, kPer = Tile<T, DP>::kPer;
    constexpr int kRows = 256 / kPieces;  // rows a pass
    constexpr int kPasses = NG * 16 / kRows;
    static_assert(kRows <= 16 || kRows % 16 == 0, "a pass covers whole groups or a part of one");
    const int tid = opaque((int)threadIdx.x);
    const int at = tid % kPieces, r0 = tid / kPieces;
#pragma unroll
    for (int i = 0; i < kPasses; i++) {
        const int r = r0 + i * kRows, y0 = i * kRows / 16;
        const int c = (at ^ (r & Tile<T, DP>::kSwizzle)) * kPer;
        long long o;
        int n;
        if constexpr (WIDE) {
            o = off[0] + (long long)r * stride + c;
            n = s.left[0] - (r & ~15);
        } else {
            o = off[y0];
            n = s.left[y0];
#pragma unroll
            for (int z = 1; z < kRows / 16; z++)
                if (r0 >> 4 == z) {
                    o = off[y0 + z];
                    n = s.left[y0 + z];
                }
            o += (long long)(r & 15) * stride + c;
        }
        fetch(t + i * 256 + uniform(tid & ~63), p + o, (r & 15) < n && c < head_dim);
    }
}

// A run of products whose operands come from LDS: AHEAD operands are on their way before the first product, and the next ones are
// asked for after every STEP, so that no product waits for the read just before it.  The fences keep the compiler from
// putting each read back before its use.
template <class F, int N, int AHEAD, int STEP, class Load, class Use> __device__ inline void pipelined(Load load, Use use)
{
    F f[AHEAD];
#pragma unroll
    for (int i = 0; i < AHEAD; i++) f[i] = load(i);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < N; i += STEP) {
#pragma unroll
        for (int s = 0; s < STEP; s++) use(i + s, f[(i + s) % AHEAD]);
#pragma unroll
        for (int s = 0; s < STEP; s++)
            if (i + s + AHEAD < N) f[(i + s) % AHEAD] = load(i + s + AHEAD);
        __builtin_amdgcn_sched_barrier(0);
    }
}

// a lane's fragments of one row: the chunks of eight columns 32 * s + 8 * quad
template <class T, int KS, bool FULL> __device__ inline void row_frags(Frag<T> (&f)[KS], const T *p, int quad, int head_dim, bool live)
{
#pragma unroll
    for (int s = 0; s < KS; s++) {
        const int d = 32 * s + 8 * quad;
        f[s] = (live && (FULL || d < head_dim)) ? frag_load(p + d) : frag_zero<T>();
    }
}

}  // namespace lm
}  // namespace nsp
