// attend_fwd.hip -- attention over the listed blocks of keys.
//
//   out[t,h] = sum_j p_j v_j,  p = softmax(scale q.k_j) over the keys j of the blocks that row (t, g) lists, g = h / group.
//
// One wavefront takes one pattern row: the group's query heads are the (up to 16) columns of its matrix products, so K and V are
// read once for all of them.  Nothing but registers: S^T = K Q^T comes out with lane l holding column (query) l % 16 and keys
// 4 (l / 16) + i, which, rounded, is already the right operand of O^T = V^T P^T; V is read row by row, E = DP / 16
// neighbouring columns a lane, and transposed inside the lane (common.h).  The softmax runs over the blocks with
// a running maximum and sum in 32 bits, in base 2.
// With few rows (a serving step) eight wavefronts share a row: wavefront w takes every eighth tile of keys and the partial
// results meet in LDS.
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
    const int g = (int)(blockIdx.x % G.kv_heads);
    const int rest = (int)(blockIdx.x / G.kv_heads);
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
            // S^T, sixteen keys at a time
            f32x4 s[NG];
#pragma unroll
            for (int y = 0; y < NG; y++) {
                const int r = col < x[y].rows ? col : 0;
                Frag<T> kf[KS];
                row_frags<T, KS, FULL>(kf, k + x[y].k_off + (long long)r * G.k_row, quad, D, true);
                s[y] = f32x4{0, 0, 0, 0};
#pragma unroll
                for (int z = 0; z < KS; z++) s[y] = mma(kf[z], qf[z], s[y]);
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
                const float alpha = exp2f(m - m_use);  // 0 while m is -inf
                l *= alpha;
#pragma unroll
                for (int j = 0; j < E; j++) o[j] *= alpha;
                m = m_new;
            }
#pragma unroll
            for (int y = 0; y < NG; y++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    s[y][e] = exp2f(s[y][e] - m_use);
                    l += s[y][e];
                }
            // O^T += V^T P^T, 32 keys at a time
#pragma unroll
            for (int y = 0; y < NG; y += 2) {
                Rows<T, E> vr;
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const Group16 &gx = x[y + (e >> 2)];
                    const int r = 4 * quad + (e & 3);
                    const T *p = v + gx.v_off + (long long)(r < gx.rows ? r : 0) * G.v_row + col * E;
                    if constexpr (FULL) rows_load(vr, e, p); else rows_load_part(vr, e, p, D - col * E);
                    // a hidden key's row must not reach the sum, whatever stands there
                    if (!whole && r >= gx.rows) rows_clear(vr, e);
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
        for (int w = 0; w < WAVES; w++) L += ml[(WAVES + w) * 16 + col] * exp2f(ml[w * 16 + col] - M_use);
        const float mine = (L == 0.f ? 0.f : 1.f / L) * exp2f(m - M_use);
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

template <class T, int DP, int NG>
static void launch_attend(const Geometry &G, const void *q, const void *k, const void *v, const int *idx, void *out, float *lse, hipStream_t st)
{
    const int slices = (int)ceil_div(G.group, 16);
    const long long rows = (long long)G.q_rows * slices;
    // eight wavefronts a row while that leaves compute units without work otherwise
    const bool split = rows * G.kv_heads < 2048;
    const bool full = G.head_dim == DP;
#define NSP_GO(FULL, WAVES)                                                                                                          \
    hipLaunchKernelGGL((k_attend<T, DP, NG, FULL, WAVES>), dim3((unsigned)((WAVES > 1 ? rows : ceil_div(G.q_rows, 4) * slices) * G.kv_heads)), \
                       dim3(WAVES > 1 ? 64 * WAVES : 256), 0, st, G, (const T *)q, (const T *)k, (const T *)v, idx, (T *)out, lse, slices)
    if (split) {
        if (full) NSP_GO(true, 8); else NSP_GO(false, 8);
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
