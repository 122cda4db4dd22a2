// common.h -- types, matrix fragments and sequence geometry of libnsparse_lm.so.
#pragma once
#include <hip/hip_runtime.h>

#include <cstdint>
#include <tuple>
#include <utility>

#include "nsparse_lm.h"

namespace nsp {
namespace lm {

// ---- errors: per thread, as codes (a C entry point never throws or aborts) -----------------------------------------
int fail(int code, const char *what);
void clear_error();
void note_launch(hipError_t e);
int launched(const char *what);  // the first error of this call's launches as a return code

// A launch whose own result counts: what other code left as the thread's last error is neither taken for ours nor taken away.
template <class... P, size_t... I>
inline void launch_packed(const void *kernel, dim3 grid, dim3 block, size_t lds, hipStream_t st, std::tuple<P...> args, std::index_sequence<I...>)
{
    void *at[] = {(void *)&std::get<I>(args)...};
    note_launch(hipLaunchKernel(kernel, grid, block, at, lds, st));
}
template <class... P, class... A> inline void launch(void (*kernel)(P...), dim3 grid, dim3 block, size_t lds, hipStream_t st, A... args)
{
    static_assert(sizeof...(P) == sizeof...(A), "an argument for every parameter");
    launch_packed((const void *)kernel, grid, block, lds, st, std::tuple<P...>(args...), std::index_sequence_for<P...>());
}

inline int elem_size(int dtype) { return dtype == NSPARSE_LM_F32 ? 4 : 2; }
constexpr long long kMostKeys = 0x7fffffffLL - 4096;  // of a sequence: a block's end is an int too
inline long long ceil_div(long long a, long long b) { return (a + b - 1) / b; }

// ---- types ---------------------------------------------------------------------------------------------------------
typedef __attribute__((ext_vector_type(4))) float f32x4;
typedef __attribute__((ext_vector_type(4))) unsigned u32x4;
typedef __attribute__((ext_vector_type(2))) unsigned u32x2;
typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;
typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;
typedef __attribute__((ext_vector_type(2))) __bf16 bf16x2;
typedef __attribute__((ext_vector_type(2))) _Float16 f16x2;

__device__ inline float to_f32(float x) { return x; }
__device__ inline float to_f32(__bf16 x) { return (float)x; }
__device__ inline float to_f32(_Float16 x) { return (float)x; }
template <class T> __device__ inline T from_f32(float x) { return (T)x; }

// two floats rounded to nearest even and packed
__device__ inline unsigned pack2(float a, float b, __bf16)
{
    bf16x2 v = {(__bf16)a, (__bf16)b};
    return __builtin_bit_cast(unsigned, v);
}
__device__ inline unsigned pack2(float a, float b, _Float16)
{
    f16x2 v = {(_Float16)a, (_Float16)b};
    return __builtin_bit_cast(unsigned, v);
}

// ---- matrix fragments -----------------------------------------------------------------------------------------------
// One fragment is a lane's share of a 16 x 32 operand of the 16 x 16 products: lane l holds row (or column) l % 16 and the
// eight contraction slots 8 * (l / 16) .. + 8.  Both operands of a product use the same slots, so any assignment of
// contraction indexes to slots is right as long as the two agree: the kernels use that to feed the output of one
// product (lane l: column l % 16, rows 4 * (l / 16) + i) straight into the next one.  Single precision does the 32
// slots as eight 16 x 16 x 4 products; 16-bit types as one 16 x 16 x 32 product.
template <class T> struct Frag { u32x4 r; };
template <> struct Frag<float> { f32x4 lo, hi; };

__device__ inline f32x4 mma(const Frag<__bf16> &a, const Frag<__bf16> &b, f32x4 c)
{
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a.r), __builtin_bit_cast(bf16x8, b.r), c, 0, 0, 0);
}
__device__ inline f32x4 mma(const Frag<_Float16> &a, const Frag<_Float16> &b, f32x4 c)
{
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a.r), __builtin_bit_cast(f16x8, b.r), c, 0, 0, 0);
}
__device__ inline f32x4 mma(const Frag<float> &a, const Frag<float> &b, f32x4 c)
{
#pragma unroll
    for (int i = 0; i < 4; i++) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.lo[i], b.lo[i], c, 0, 0, 0);
#pragma unroll
    for (int i = 0; i < 4; i++) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.hi[i], b.hi[i], c, 0, 0, 0);
    return c;
}

template <class T> __device__ inline Frag<T> frag_zero() { return Frag<T>{u32x4{0, 0, 0, 0}}; }
template <> __device__ inline Frag<float> frag_zero<float>() { return Frag<float>{f32x4{0, 0, 0, 0}, f32x4{0, 0, 0, 0}}; }

// eight neighbouring elements (16 bytes, or 32 in single precision; the host checked the alignment)
template <class T> __device__ inline Frag<T> frag_load(const T *p) { return Frag<T>{*(const u32x4 *)p}; }
template <> __device__ inline Frag<float> frag_load<float>(const float *p) { return Frag<float>{*(const f32x4 *)p, *(const f32x4 *)(p + 4)}; }

template <class T> __device__ inline void frag_negate(Frag<T> &f) { f.r ^= 0x80008000u; }
template <> __device__ inline void frag_negate<float>(Frag<float> &f)
{
    f.lo = -f.lo;
    f.hi = -f.hi;
}

template <class T> __device__ inline float frag_dot(const Frag<T> &a, const Frag<T> &b)
{
    typedef __attribute__((ext_vector_type(8))) T T8;
    T8 x = __builtin_bit_cast(T8, a.r), y = __builtin_bit_cast(T8, b.r);
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < 8; i++) s += (float)x[i] * (float)y[i];
    return s;
}
template <> __device__ inline float frag_dot<float>(const Frag<float> &a, const Frag<float> &b)
{
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < 4; i++) s += a.lo[i] * b.lo[i];
#pragma unroll
    for (int i = 0; i < 4; i++) s += a.hi[i] * b.hi[i];
    return s;
}

// Output of two 16 x 16 products (rows 4 * (l / 16) + i of each) as one fragment: slot i < 4 is row i of the first,
// slot 4 + i row i of the second.  slot_row() names the row that lane group `quad` holds in slot s.
template <class T> __device__ inline Frag<T> frag_pack(f32x4 a, f32x4 b)
{
    T t{};
    return Frag<T>{u32x4{pack2(a[0], a[1], t), pack2(a[2], a[3], t), pack2(b[0], b[1], t), pack2(b[2], b[3], t)}};
}
template <> __device__ inline Frag<float> frag_pack<float>(f32x4 a, f32x4 b) { return Frag<float>{a, b}; }

// the same, half by half
template <class T> __device__ inline void frag_half(Frag<T> &f, int h, f32x4 a)
{
    f.r[2 * h] = pack2(a[0], a[1], T{});
    f.r[2 * h + 1] = pack2(a[2], a[3], T{});
}
template <> __device__ inline void frag_half<float>(Frag<float> &f, int h, f32x4 a)
{
    if (h == 0) f.lo = a; else f.hi = a;
}

// ---- a lane's share of 8 rows x E columns, and the E fragments of its transpose --------------------------------------
// Lane (quad, r) loads, of each of its quad's eight slot rows, the E = DP / 16 neighbouring columns r * E ..: a row is read
// by 16 lanes in one piece.  Fragment j of the transpose has column r * E + j as its row: which column a product's
// row stands for is free as well, and the output of a lane is then E neighbouring columns again.
template <class T, int E> struct Rows { unsigned w[8][E / 2]; };
template <int E> struct Rows<float, E> { float w[8][E]; };

template <class T, int E> __device__ inline void rows_load(Rows<T, E> &x, int s, const T *p)
{
    if constexpr (E == 4) {
        u32x2 v = *(const u32x2 *)p;
        x.w[s][0] = v[0];
        x.w[s][1] = v[1];
    } else {
#pragma unroll
        for (int c = 0; c < E / 8; c++) {
            u32x4 v = *(const u32x4 *)(p + 8 * c);
#pragma unroll
            for (int i = 0; i < 4; i++) x.w[s][4 * c + i] = v[i];
        }
    }
}
template <int E> __device__ inline void rows_load(Rows<float, E> &x, int s, const float *p)
{
#pragma unroll
    for (int c = 0; c < E / 4; c++) {
        f32x4 v = *(const f32x4 *)(p + 4 * c);
#pragma unroll
        for (int i = 0; i < 4; i++) x.w[s][4 * c + i] = v[i];
    }
}
template <class T, int E> __device__ inline void rows_clear(Rows<T, E> &x, int s)
{
#pragma unroll
    for (int i = 0; i < (int)(sizeof(x.w[s]) / sizeof(x.w[s][0])); i++) x.w[s][i] = 0;
}
// the first `n` of the E columns exist (n a multiple of 4 for E = 4, of 8 else; the others read as 0)
template <class T, int E> __device__ inline void rows_load_part(Rows<T, E> &x, int s, const T *p, int n)
{
    if (n >= E) {
        rows_load(x, s, p);
        return;
    }
    rows_clear(x, s);
    if constexpr (E == 16) {
        if (n >= 8) {
            Rows<T, 8> h;
            rows_load(h, 0, p);
#pragma unroll
            for (int i = 0; i < (int)(sizeof(h.w[0]) / sizeof(h.w[0][0])); i++) x.w[s][i] = h.w[0][i];
        }
    }
}
template <class T, int E> __device__ inline Frag<T> rows_column(const Rows<T, E> &x, int j)
{
    const unsigned sel = (j & 1) ? 0x07060302u : 0x05040100u;
    const int w = j >> 1;
    return Frag<T>{u32x4{__builtin_amdgcn_perm(x.w[1][w], x.w[0][w], sel), __builtin_amdgcn_perm(x.w[3][w], x.w[2][w], sel),
                         __builtin_amdgcn_perm(x.w[5][w], x.w[4][w], sel), __builtin_amdgcn_perm(x.w[7][w], x.w[6][w], sel)}};
}
template <int E> __device__ inline Frag<float> rows_column(const Rows<float, E> &x, int j)
{
    return Frag<float>{f32x4{x.w[0][j], x.w[1][j], x.w[2][j], x.w[3][j]}, f32x4{x.w[4][j], x.w[5][j], x.w[6][j], x.w[7][j]}};
}

// E neighbouring columns of an output row
template <class T, int E> __device__ inline void store_columns(T *p, const float *v, int n)
{
    if (n <= 0) return;
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int c = 0; c < E / 4; c++)
            if (4 * c < n) *(f32x4 *)(p + 4 * c) = f32x4{v[4 * c], v[4 * c + 1], v[4 * c + 2], v[4 * c + 3]};
    } else if constexpr (E == 4) {
        *(u32x2 *)p = u32x2{pack2(v[0], v[1], T{}), pack2(v[2], v[3], T{})};
    } else {
#pragma unroll
        for (int c = 0; c < E / 8; c++)
            if (8 * c < n)
                *(u32x4 *)(p + 8 * c) = u32x4{pack2(v[8 * c], v[8 * c + 1], T{}), pack2(v[8 * c + 2], v[8 * c + 3], T{}),
                                              pack2(v[8 * c + 4], v[8 * c + 5], T{}), pack2(v[8 * c + 6], v[8 * c + 7], T{})};
    }
}

// ---- lanes ---------------------------------------------------------------------------------------------------------
__device__ inline int lane_id() { return (int)(threadIdx.x & 63); }
__device__ inline int read_lane(int v, int lane) { return __builtin_amdgcn_readlane(v, lane); }
__device__ inline long long read_lane64(long long v, int lane)
{
    const unsigned lo = (unsigned)read_lane((int)v, lane), hi = (unsigned)read_lane((int)(v >> 32), lane);
    return (long long)(((unsigned long long)hi << 32) | lo);
}
// over the four lane groups that share a column of a product's output
__device__ inline float quads_max(float x)
{
    auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
    r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ inline float quads_sum(float x)
{
    auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
// x, which the compiler cannot know: what depends on it is computed where it is used and not kept in registers over a loop
__device__ inline int opaque(int x)
{
    asm volatile("" : "+v"(x));
    return x;
}
// v of another lane
__device__ inline int pull(int v, int lane) { return __builtin_amdgcn_ds_bpermute(lane << 2, v); }
__device__ inline int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ inline unsigned long long uniform64(unsigned long long v)
{
    return ((unsigned long long)(unsigned)uniform((int)(v >> 32)) << 32) | (unsigned)uniform((int)v);
}
// over the wavefront, the result everywhere: inside the rows of sixteen by their neighbours, then over the four rows
__device__ inline float wave_max(float x)
{
    x = fmaxf(x, __uint_as_float(__builtin_amdgcn_mov_dpp(__float_as_uint(x), 0xb1, 0xf, 0xf, false)));
    x = fmaxf(x, __uint_as_float(__builtin_amdgcn_mov_dpp(__float_as_uint(x), 0x4e, 0xf, 0xf, false)));
    x = fmaxf(x, __uint_as_float(__builtin_amdgcn_mov_dpp(__float_as_uint(x), 0x141, 0xf, 0xf, false)));
    x = fmaxf(x, __uint_as_float(__builtin_amdgcn_mov_dpp(__float_as_uint(x), 0x140, 0xf, 0xf, false)));
    return quads_max(x);
}

// 2^x in one instruction; what is below 2^-126 becomes 0, which no sum next to a 1 can tell
__device__ inline float pow2(float x) { return __builtin_amdgcn_exp2f(x); }

// ---- geometry of a call ------------------------------------------------------------------------------------------------
struct Geometry {
    int n_seq, heads, kv_heads, group, head_dim, block, width, causal, page_size, per_page;
    int q_rows, q_each;            // q_each: query rows a sequence without cu_q
    long long k_rows, k_each;      // k_each: key rows a sequence without cu_k
    long long table_stride;
    int blocks_each;               // mean rows a sequence without cu_k
    const int *cu_q, *cu_k, *q_len, *k_len, *page_table;
    long long q_row, q_head, k_page, k_row, k_head, v_page, v_row, v_head;
    float scale;
};
int geometry(const nsparse_lm_attn *a, bool needs_q, bool needs_k, Geometry *g);  // checks the arguments

struct Seq {
    int s;            // sequence
    int q_len, k_len; // rows that count
    int q_end;        // of a query row's sequence: from that row up to here every row is the sequence's
    long long q_base; // first query row
    long long k_base; // first key row (not paged)
};

__device__ inline int clampi(int x, int lo, int hi) { return x < lo ? lo : (x > hi ? hi : x); }

__device__ inline Seq seq_at(const Geometry &G, int s)
{
    Seq q;
    q.s = s;
    q.q_end = 0;
    if (G.cu_q) {
        const int a = clampi(G.cu_q[s], 0, G.q_rows), b = clampi(G.cu_q[s + 1], a, G.q_rows);
        q.q_base = a;
        q.q_len = b - a;
    } else {
        q.q_base = (long long)s * G.q_each;
        q.q_len = G.q_each;
    }
    if (G.q_len) q.q_len = clampi(G.q_len[s], 0, q.q_len);
    long long cap;
    if (G.page_size > 0) {
        q.k_base = 0;
        cap = G.k_rows > 0 ? G.table_stride * G.page_size : 0;
    } else if (G.cu_k) {
        const int hi = (int)G.k_rows;
        const int a = clampi(G.cu_k[s], 0, hi), b = clampi(G.cu_k[s + 1], a, hi);
        q.k_base = a;
        cap = b - a;
    } else {
        q.k_base = (long long)s * G.k_each;
        cap = G.k_each;
    }
    if (cap > kMostKeys) cap = kMostKeys;
    q.k_len = G.k_len ? clampi(G.k_len[s], 0, (int)cap) : (int)cap;
    return q;
}

// Workgroups of a launch, counted through both dimensions of the grid: one dimension holds less than 2^32 threads.  There may be up
// to kGridX - 1 more of them than asked for.
constexpr long long kGridX = 1 << 21, kMostGroups = 0x7fffffffLL - kGridX;
inline dim3 groups(long long n) { return n <= kGridX ? dim3((unsigned)n) : dim3((unsigned)kGridX, (unsigned)ceil_div(n, kGridX)); }
__device__ inline unsigned group_id() { return blockIdx.y * gridDim.x + blockIdx.x; }

// the sequence of query row t and the row's number inside it, or -1 where no sequence has it.  Where cu_q does not ascend the search still
// decides whose a row is: a number that it finds above t ends the rows that it decides alike.
__device__ inline int seq_of_query(const Geometry &G, int t, Seq &q)
{
    int s, end = G.q_rows;
    if (G.cu_q) {
        const int last = G.cu_q[G.n_seq];
        if (t >= last || t < G.cu_q[0]) return -1;
        end = last < end ? last : end;
        int lo = 0, hi = G.n_seq;  // the last s with cu_q[s] <= t
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1, c = G.cu_q[mid];
            if (c <= t) {
                lo = mid;
            } else {
                hi = mid;
                end = c < end ? c : end;
            }
        }
        s = lo;
    } else {
        s = t / G.q_each;
    }
    q = seq_at(G, s);
    q.q_end = q.q_base + q.q_len < end ? (int)(q.q_base + q.q_len) : end;
    const long long i = (long long)t - q.q_base;
    return (i >= 0 && i < q.q_len) ? (int)i : -1;
}

// mean row of block 0 of a sequence (not paged)
__device__ inline long long mean_base(const Geometry &G, const Seq &q)
{
    return G.cu_k ? q.k_base / G.block + q.s : (long long)q.s * G.blocks_each;
}
// sequence and block of a mean row (not paged); false where the row belongs to no block
__device__ inline bool block_of_mean_row(const Geometry &G, long long row, Seq &q, int &b)
{
    int s;
    if (G.cu_k) {
        int lo = 0, hi = G.n_seq;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if ((long long)G.cu_k[mid] / G.block + mid <= row) lo = mid; else hi = mid;
        }
        s = lo;
    } else {
        s = (int)(row / G.blocks_each);
    }
    if (s >= G.n_seq) return false;
    q = seq_at(G, s);
    const long long d = row - mean_base(G, q);
    b = (int)d;
    return d >= 0 && d * G.block < q.k_len;
}
// page of block b of a paged sequence, -1 where the table names none
__device__ inline long long page_of_block(const Geometry &G, int s, int b)
{
    const int p = G.page_table[(long long)s * G.table_stride + b / G.per_page];
    return (p < 0 || p >= G.k_rows) ? -1 : p;
}

// ---- a pattern row ---------------------------------------------------------------------------------------------------
// Up to 64 entries at a time: lane i reads entry at + i, entries that do not count are dropped (see the header: not negative,
// inside `blocks`, greater than all before), and the ones that count are moved to the first lanes.
// `seen` carries the greatest entry of the row so far.  Returns how many; `block` is lane i's entry.
__device__ inline int pattern_chunk(const int *row, int at, int width, int blocks, int &seen, int &block)
{
    const int lane = opaque(lane_id());
    const int e = at + lane < width ? row[at + lane] : -1;
    int top = e;  // greatest entry up to and including this lane
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int o = pull(top, lane - d);
        if (lane >= d) top = top > o ? top : o;
    }
    int before = pull(top, lane - 1);
    before = lane == 0 ? seen : (before > seen ? before : seen);
    const bool counts = e >= 0 && e < blocks && e > before;
    const unsigned long long mask = __ballot(counts);
    const int last = read_lane(top, 63);
    seen = last > seen ? last : seen;
    const int n = __popcll(mask);
    const unsigned long long below = (1ULL << lane) - 1;
    const int dst = counts ? __popcll(mask & below) : n + __popcll(~mask & below);
    block = __builtin_amdgcn_ds_permute(dst << 2, e);
    return n;
}

}  // namespace lm
}  // namespace nsp
