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
// Bound by reading K once.
template <class T>
__global__ void __launch_bounds__(256) k_block_means(const Geometry G, const T *__restrict__ k, T *__restrict__ means, int last, int per_seq)
{
    __shared__ double part[256 * 8];
    const int g = (int)(blockIdx.x % G.kv_heads);
    const long long rest = blockIdx.x / G.kv_heads;
    Seq sq;
    int b;
    if (per_seq > 0) {
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
// One workgroup per (query row, key head): the scores of `kScores` blocks at a time in LDS beside the best so far, the best of
// both by repeated search.
constexpr int kScores = 4096, kWidest = 256;

template <class T>
__global__ void __launch_bounds__(256)
    k_select(const Geometry G, int first, int local, const T *__restrict__ q, const T *__restrict__ means, int *__restrict__ idx)
{
    __shared__ double qsum[256];
    __shared__ double score[kScores + kWidest];
    __shared__ int name[kScores + kWidest];
    __shared__ double wave_best[4];
    __shared__ int wave_at[4];
    __shared__ double best_score[kWidest];
    __shared__ int best_name[kWidest];
    const int g = (int)(blockIdx.x % G.kv_heads), t = (int)(blockIdx.x / G.kv_heads);
    const int tid = threadIdx.x;
    Seq sq;
    const int i = seq_of_query(G, t, sq);
    if (i < 0) return;
    int eligible;  // blocks 0 .. eligible - 1
    if (G.causal) {
        const int pos = sq.k_len - sq.q_len + i;
        eligible = pos < 0 ? 0 : pos / G.block + 1;
    } else {
        eligible = (sq.k_len + G.block - 1) / G.block;
    }
    int *row = idx + ((long long)t * G.kv_heads + g) * G.width;
    if (eligible <= G.width) {
        for (int x = tid; x < G.width; x += 256) row[x] = x < eligible ? x : -1;
        return;
    }
    const int lo = first, hi = eligible - local;  // the blocks that compete; eligible > width >= first + local
    const int need = G.width - first - local;
    for (int d = tid; d < G.head_dim; d += 256) {
        double s = 0;
        for (int h = 0; h < G.group; h++) s += (double)to_f32(q[(long long)t * G.q_row + (long long)(g * G.group + h) * G.q_head + d]);
        qsum[d] = s;
    }
    __syncthreads();
    int have = 0;
    for (int c0 = lo; c0 < hi && need > 0; c0 += kScores) {
        const int n = hi - c0 < kScores ? hi - c0 : kScores;
        for (int x = tid; x < have; x += 256) {
            score[x] = best_score[x];
            name[x] = best_name[x];
        }
        for (int x = tid; x < n; x += 256) {
            const int b = c0 + x;
            long long m;
            if (G.page_size > 0) {
                const long long page = page_of_block(G, sq.s, b);
                m = page < 0 ? -1 : page * G.per_page + b % G.per_page;
            } else {
                m = mean_base(G, sq) + b;
            }
            double s = -INFINITY;
            if (m >= 0) {
                const T *p = means + (m * G.kv_heads + g) * G.head_dim;
                s = 0;
                for (int d = 0; d < G.head_dim; d++) s += qsum[d] * (double)to_f32(p[d]);
                if (s != s) s = -INFINITY;
            }
            score[have + x] = s;
            name[have + x] = b;
        }
        __syncthreads();
        const int total = have + n;
        const int take = need < total ? need : total;
        for (int r = 0; r < take; r++) {
            double bs = -INFINITY;
            int bn = 0x7fffffff, at = -1;
            for (int x = tid; x < total; x += 256)
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
            if ((tid & 63) == 0) {
                wave_best[tid >> 6] = bs;
                wave_at[tid >> 6] = at;
            }
            __syncthreads();
            if (tid == 0) {
                int pick = -1;
                for (int w = 0; w < 4; w++) {
                    const int a = wave_at[w];
                    if (a < 0) continue;
                    if (pick < 0 || wave_best[w] > score[pick] || (wave_best[w] == score[pick] && name[a] < name[pick])) pick = a;
                }
                best_score[r] = score[pick];
                best_name[r] = name[pick];
                name[pick] = -1;
            }
            __syncthreads();
        }
        have = take;
    }
    for (int x = tid; x < first; x += 256) row[x] = x;
    for (int x = tid; x < local; x += 256) row[G.width - local + x] = hi + x;
    for (int x = tid; x < have; x += 256) {
        int r = 0;
        for (int y = 0; y < have; y++) r += best_name[y] < best_name[x];
        row[first + r] = best_name[x];
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
    if (last > 0) per_seq = (last - 1) / G.block + 2;
    if (G.page_size > 0 && (per_seq == 0 || per_seq > G.table_stride * G.per_page)) per_seq = G.table_stride * G.per_page;
    rows = per_seq > 0 ? per_seq * G.n_seq : nsparse_lm_mean_rows(a);
    if (rows * G.kv_heads > 0x7fffffffLL) return fail(NSPARSE_LM_EARG, "block_means: blocks x heads out of range");
    if (rows == 0) return 0;
    const dim3 grid((unsigned)(rows * G.kv_heads));
    hipStream_t st = (hipStream_t)stream;
    if (a->dtype == NSPARSE_LM_BF16)
        hipLaunchKernelGGL(k_block_means<__bf16>, grid, dim3(256), 0, st, G, (const __bf16 *)k, (__bf16 *)means, last, (int)per_seq);
    else if (a->dtype == NSPARSE_LM_F16)
        hipLaunchKernelGGL(k_block_means<_Float16>, grid, dim3(256), 0, st, G, (const _Float16 *)k, (_Float16 *)means, last, (int)per_seq);
    else
        hipLaunchKernelGGL(k_block_means<float>, grid, dim3(256), 0, st, G, (const float *)k, (float *)means, last, (int)per_seq);
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
    const dim3 grid((unsigned)((long long)G.q_rows * G.kv_heads));
    hipStream_t st = (hipStream_t)stream;
    if (a->dtype == NSPARSE_LM_BF16)
        hipLaunchKernelGGL(k_select<__bf16>, grid, dim3(256), 0, st, G, a->first, a->local, (const __bf16 *)q, (const __bf16 *)means, idx);
    else if (a->dtype == NSPARSE_LM_F16)
        hipLaunchKernelGGL(k_select<_Float16>, grid, dim3(256), 0, st, G, a->first, a->local, (const _Float16 *)q, (const _Float16 *)means, idx);
    else
        hipLaunchKernelGGL(k_select<float>, grid, dim3(256), 0, st, G, a->first, a->local, (const float *)q, (const float *)means, idx);
    return launched("select_blocks");
}
}
