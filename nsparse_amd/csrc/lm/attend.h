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
// The rows of neighbouring queries list mostly the same blocks.  A wavefront that has several of them walks the union of their
// rows, block by block upwards: lane i < 32 is a cursor on row i (the entries that count ascend, see the header), the least head is
// the next block, the lanes whose head it is are the queries that list it.
struct Cursors {
    const int *row;
    int at, width;   // next entry, entries
    int ahead;       // entry `at`, fetched early
    int seen, head;  // greatest entry so far; the next that counts, kNone behind the last
    int blocks;      // blocks with keys that this row's query sees
};
constexpr int kNone = 0x7fffffff;

__device__ inline void cursor_advance(Cursors &c)
{
    c.head = kNone;
    while (c.at < c.width) {
        const int e = c.ahead;
        if (++c.at < c.width) c.ahead = c.row[c.at];
        if (e > c.seen) {
            c.seen = e;
            if (e < c.blocks) c.head = e; else c.at = c.width;  // all that could count behind it is greater still
            break;
        }
    }
}
__device__ inline Cursors cursor_open(const int *row, int width, int blocks, bool live)
{
    Cursors c;
    c.row = row;
    c.width = (live && blocks > 0) ? width : 0;
    c.at = 0;
    c.seen = -1;
    c.blocks = blocks;
    c.ahead = c.width > 0 ? row[0] : -1;
    cursor_advance(c);
    return c;
}
// the next block of the union and the lanes that list it; kNone at the end
__device__ inline int cursors_next(Cursors &c, unsigned &who)
{
    const int b = least_of_32(c.head);
    const bool mine = c.head == b;
    who = (unsigned)__ballot(mine);
    if (b == kNone) return kNone;
    if (mine) cursor_advance(c);
    return b;
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
