// route.hip -- tokens sorted by expert, and back with weights.
//
// The router's choice is a tokens x experts matrix with `top` entries a row.  Sorting its entries by expert (stable) is the
// transposition of that matrix: count per chunk of entries, prefix sums per expert, then every entry finds its row as
//   rows of smaller experts + the expert's rows of earlier chunks + of earlier wavefronts + of earlier lanes,
// each a count of what stands before it, so no atomic decides an order.  The products with the matrix are one pass over the token
// rows; every kernel works token by token: the token's row stays in registers or cache while its `top` rows are read or written.
// All of it is bound by memory: gather and combine of 16384 x 4096 bf16 rows, 8 entries each, 250 and 272 us, the gradient of combine 462 (1.2, 1.2
// and 2.3 GB; a large copy reaches 4.8 TB/s); sorting 131072 entries 13 us in three launches, up to 4096 entries 6 us in one.
#include "common.h"

namespace nsp {
namespace lm {

constexpr int kPerWave = 256;  // entries a wavefront of the sort: four rounds of 64
constexpr int kMaxExperts = 4096;

// wavefronts a workgroup: their counters, 2 bytes an expert each, take at most 32 KB of LDS
inline int sort_waves(int experts) { return experts <= 1024 ? 16 : experts <= 2048 ? 8 : 4; }

// lanes with the same number as this one, among those with `in`
__device__ inline unsigned long long same_lanes(int id, bool in, int bits)
{
    unsigned long long m = __ballot(in);
    for (int b = 0; b < bits; b++) {
        const unsigned long long set = __ballot((id >> b) & 1);
        m &= ((id >> b) & 1) ? set : ~set;
    }
    return m;
}

__global__ void __launch_bounds__(1024) k_route_count(const int *__restrict__ ids, int n, int experts, int *__restrict__ counts)
{
    extern __shared__ int hist[];
    const int per = (int)(blockDim.x >> 6) * kPerWave;
    for (int e = threadIdx.x; e < experts; e += blockDim.x) hist[e] = 0;
    __syncthreads();
    const int a = (int)blockIdx.x * per, z = n - a < per ? n : a + per;
    for (int x = a + (int)threadIdx.x; x < z; x += blockDim.x) {
        const int id = ids[x];
        if (id >= 0 && id < experts) atomicAdd(&hist[id], 1);
    }
    __syncthreads();
    for (int e = threadIdx.x; e < experts; e += blockDim.x) counts[(long long)blockIdx.x * experts + e] = hist[e];
}

// counts[c][e] -> rows of expert e in the chunks before c; total[e] = all of them.  One wavefront an expert.
__global__ void __launch_bounds__(64) k_route_prefix(int *__restrict__ counts, int *__restrict__ total, int chunks, int experts)
{
    const int e = blockIdx.x, lane = lane_id();
    int run = 0;
    for (int c0 = 0; c0 < chunks; c0 += 64) {
        const int c = c0 + lane;
        const int v = c < chunks ? counts[(long long)c * experts + e] : 0;
        int s = v;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int o = __shfl_up(s, d);
            if (lane >= d) s += o;
        }
        if (c < chunks) counts[(long long)c * experts + e] = run + s - v;
        run += read_lane(s, 63);
    }
    if (lane == 0) total[e] = run;
}

// ONE: the only chunk, no counts from other kernels
template <bool ONE>
__global__ void __launch_bounds__(1024)
    k_route_place(const int *__restrict__ ids, int n, int experts, int bits, const int *__restrict__ counts, const int *__restrict__ total,
                  int *__restrict__ offsets, int *__restrict__ order, int *__restrict__ place)
{
    extern __shared__ int lds[];
    int *start = lds;                                          // experts: first row of the expert in this chunk
    unsigned short *before = (unsigned short *)(lds + experts);  // waves x experts
    __shared__ int wave_sum[16];
    const int lane = lane_id(), waves = (int)(blockDim.x >> 6);
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    unsigned short *mine = before + wave * experts;
    for (int x = threadIdx.x; x < waves * experts; x += blockDim.x) before[x] = 0;
    __syncthreads();
    const int a = (int)blockIdx.x * waves * kPerWave + wave * kPerWave;
    int id[kPerWave / 64], rank[kPerWave / 64];
#pragma unroll
    for (int r = 0; r < kPerWave / 64; r++) {
        const long long x = (long long)a + 64 * r + lane;
        id[r] = x < n ? ids[x] : -1;
        if (id[r] < 0 || id[r] >= experts) id[r] = -1;
        const unsigned long long same = same_lanes(id[r], id[r] >= 0, bits);
        const int below = __popcll(same & ((1ULL << lane) - 1));
        rank[r] = 0;
        if (id[r] >= 0) {
            const int had = mine[id[r]];
            rank[r] = had + below;
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
            if (below == 0) mine[id[r]] = (unsigned short)(had + __popcll(same));
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }
    __syncthreads();
    // per expert: what the wavefronts before have, and the rows of the smaller experts (a scan over all of them)
    int carry = 0;
    for (int e0 = 0; e0 < experts; e0 += blockDim.x) {
        const int e = e0 + (int)threadIdx.x;
        int all = 0;
        if (e < experts) {
            for (int w = 0; w < waves; w++) {
                const int c = before[w * experts + e];
                before[w * experts + e] = (unsigned short)all;
                all += c;
            }
            if (!ONE) all = total[e];
        }
        int s = all;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int o = __shfl_up(s, d);
            if (lane >= d) s += o;
        }
        if (lane == 63) wave_sum[wave] = s;
        __syncthreads();
        int base = carry;
        for (int w = 0; w < waves; w++) {
            if (w < wave) base += wave_sum[w];
            carry += wave_sum[w];
        }
        if (e < experts) {
            start[e] = base + s - all + (ONE ? 0 : counts[(long long)blockIdx.x * experts + e]);
            if (blockIdx.x == 0) offsets[e] = base + s - all;
        }
        __syncthreads();
    }
    if (blockIdx.x == 0 && threadIdx.x == 0) offsets[experts] = carry;
#pragma unroll
    for (int r = 0; r < kPerWave / 64; r++) {
        const long long x = (long long)a + 64 * r + lane;
        if (x >= n) continue;
        int p = -1;
        if (id[r] >= 0) {
            p = start[id[r]] + mine[id[r]] + rank[r];
            order[p] = (int)x;
        }
        place[x] = p;
    }
}

// ---- products with the routing matrix -----------------------------------------------------------------------------------
// A row is read in pieces of 16 bytes, V elements, the last one element by element where it is shorter.  Rows of odd sizes begin at any element:
// memory takes pieces from there too (1003 fp32 rows of 1023, 3 entries each, against element by element: combine 6 and 10 us, gather 5 and 7).
template <class T> struct Piece {
    static constexpr int V = 16 / (int)sizeof(T);
    typedef __attribute__((ext_vector_type(V))) T Vec;
    struct __attribute__((packed, aligned(sizeof(T)))) Loose { Vec v; };
    static __device__ inline Vec load(const T *p, int n)
    {
        if (n >= V) return ((const Loose *)p)->v;
        Vec v{};
#pragma unroll
        for (int i = 0; i < V; i++)
            if (i < n) v[i] = p[i];
        return v;
    }
    static __device__ inline void store(T *p, const Vec &v, int n)
    {
        if (n >= V) {
            ((Loose *)p)->v = v;
            return;
        }
#pragma unroll
        for (int i = 0; i < V; i++)
            if (i < n) p[i] = v[i];
    }
    static __device__ inline Vec round(const float (&x)[V])
    {
        Vec v;
#pragma unroll
        for (int i = 0; i < V; i++) v[i] = from_f32<T>(x[i]);
        return v;
    }
};

// U: an unsigned type of the elements' size, moved as bits
template <class U>
__global__ void __launch_bounds__(256)
    k_gather_tokens(const U *__restrict__ x, const int *__restrict__ place, int tokens, int top, int channels, int per, U *__restrict__ xs)
{
    const unsigned t = group_id() * (256 / per) + threadIdx.x / per;
    if (t >= (unsigned)tokens) return;
    const int *pl = place + (long long)t * top;
    const unsigned rows = (unsigned)tokens * top;
    for (int c = ((int)threadIdx.x % per) * Piece<U>::V; c < channels; c += per * Piece<U>::V) {
        const auto v = Piece<U>::load(x + (long long)t * channels + c, channels - c);
        for (int j = 0; j < top; j++) {
            const int p = pl[j];
            if ((unsigned)p < rows) Piece<U>::store(xs + (long long)p * channels + c, v, channels - c);
        }
    }
}

template <class T>
__global__ void __launch_bounds__(256)
    k_combine_tokens(const T *__restrict__ y, const int *__restrict__ place, const float *__restrict__ w, int tokens, int top, int channels,
                     int per, T *__restrict__ out)
{
    constexpr int V = Piece<T>::V;
    const unsigned t = group_id() * (256 / per) + threadIdx.x / per;
    if (t >= (unsigned)tokens) return;
    const long long e0 = (long long)t * top;
    const unsigned rows = (unsigned)tokens * top;
    for (int c = ((int)threadIdx.x % per) * V; c < channels; c += per * V) {
        float a[V] = {};
#pragma unroll 4
        for (int j = 0; j < top; j++) {
            const int p = place[e0 + j];
            if ((unsigned)p >= rows) continue;
            const auto x = Piece<T>::load(y + (long long)p * channels + c, channels - c);
            const float f = w ? w[e0 + j] : 1.f;
#pragma unroll
            for (int i = 0; i < V; i++) a[i] += f * (float)x[i];
        }
        Piece<T>::store(out + (long long)t * channels + c, Piece<T>::round(a), channels - c);
    }
}

template <class T>
__global__ void __launch_bounds__(256)
    k_combine_tokens_bwd(const T *__restrict__ dout, const T *__restrict__ y, const int *__restrict__ place, const float *__restrict__ w,
                         int tokens, int top, int channels, int per, T *__restrict__ dy, float *__restrict__ dw)
{
    constexpr int V = Piece<T>::V;
    constexpr int J = 4;  // entries at a time: their rows are on their way together, dout is read once for them
    __shared__ float sums[2][4][J];
    const unsigned t = group_id() * (256 / per) + threadIdx.x / per;
    if (t >= (unsigned)tokens) return;  // whole wavefronts; with per = 256 the whole workgroup
    const long long e0 = (long long)t * top;
    const T *g = dout + (long long)t * channels;
    for (int j0 = 0; j0 < top; j0 += J) {
        int p[J];
        float f[J], dot[J];
#pragma unroll
        for (int j = 0; j < J; j++) {
            const bool in = j0 + j < top;
            p[j] = in ? place[e0 + j0 + j] : -1;
            if ((unsigned)p[j] >= (unsigned)tokens * top) p[j] = -1;
            f[j] = in && w ? w[e0 + j0 + j] : 1.f;
            dot[j] = 0.f;
        }
        for (int c = ((int)threadIdx.x % per) * V; c < channels; c += per * V) {
            const auto a = Piece<T>::load(g + c, channels - c);
            typename Piece<T>::Vec x[J];
#pragma unroll
            for (int j = 0; j < J; j++) {
                x[j] = typename Piece<T>::Vec{};
                if (dw && p[j] >= 0) x[j] = Piece<T>::load(y + (long long)p[j] * channels + c, channels - c);
            }
#pragma unroll
            for (int j = 0; j < J; j++) {
                if (p[j] < 0) continue;
                float b[V];
#pragma unroll
                for (int i = 0; i < V; i++) {
                    dot[j] += (float)a[i] * (float)x[j][i];
                    b[i] = (float)a[i] * f[j];
                }
                Piece<T>::store(dy + (long long)p[j] * channels + c, Piece<T>::round(b), channels - c);
            }
        }
        if (!dw) continue;
#pragma unroll
        for (int j = 0; j < J; j++)
#pragma unroll
            for (int d = 32; d > 0; d >>= 1) dot[j] += __shfl_xor(dot[j], d);
        const int left = top - j0 < J ? top - j0 : J;
        float(*part)[J] = sums[(j0 / J) & 1];  // the other half is free until the next entries
        if (per == 64) {
#pragma unroll
            for (int j = 0; j < J; j++)
                if (lane_id() == j && j < left) dw[e0 + j0 + j] = dot[j];
        } else {
#pragma unroll
            for (int j = 0; j < J; j++)
                if (lane_id() == j) part[threadIdx.x >> 6][j] = dot[j];
            __syncthreads();
            const int j = (int)threadIdx.x;
            if (j < left) dw[e0 + j0 + j] = part[0][j] + part[1][j] + part[2][j] + part[3][j];
        }
    }
}

static int check_products(int dtype, long long tokens, int top, int channels, const char *what)
{
    if (dtype != NSPARSE_LM_F32 && dtype != NSPARSE_LM_F16 && dtype != NSPARSE_LM_BF16) return fail(NSPARSE_LM_ETYPE, "dtype is none of F32, F16, BF16");
    if (tokens < 0 || top < 1 || channels < 1 || channels > 1 << 28 || tokens > (0x7fffffffLL - 4096) / top) return fail(NSPARSE_LM_EARG, what);
    return 0;
}
// threads a token: a wavefront for rows of at most 2 KB, whose pieces leave half a workgroup without work, else a workgroup.  Gradient of
// combine, bf16, by wavefront against by workgroup: 16384 tokens of 1024 channels, 4 entries each: 52 and 69 us, of 512: 27 and 44; 8192 of
// 2048: 59 and 53, of 4096: 141 and 129; 256 of 4096, 8 entries each: 25 and 10.
static int threads_per_token(int channels, int dtype) { return (long long)channels * elem_size(dtype) <= 2048 ? 64 : 256; }

}  // namespace lm
}  // namespace nsp

extern "C" {

long long nsparse_lm_route_workspace(long long tokens, int top, int experts)
{
    using namespace nsp::lm;
    clear_error();
    if (tokens < 0 || top < 1 || experts < 1 || experts > kMaxExperts || tokens > (0x7fffffffLL - 4096) / top)
        return fail(NSPARSE_LM_EARG, "route: tokens, top or experts out of range");
    const long long chunks = ceil_div(tokens * top, sort_waves(experts) * kPerWave);
    return chunks <= 1 ? 0 : 4 * (chunks + 1) * experts;
}

int nsparse_lm_route(const int *ids, long long tokens, int top, int experts, int *offsets, int *order, int *place, void *workspace,
                     long long workspace_bytes, void *stream)
{
    using namespace nsp::lm;
    const long long need = nsparse_lm_route_workspace(tokens, top, experts);
    if (need < 0) return (int)need;
    const int n = (int)(tokens * top);
    if (!offsets || (n > 0 && (!ids || !order || !place))) return fail(NSPARSE_LM_EARG, "route: a required pointer is NULL");
    if (need > 0 && (!workspace || workspace_bytes < need))
        return fail(NSPARSE_LM_EWORKSPACE, "route: workspace smaller than nsparse_lm_route_workspace() says");
    hipStream_t st = (hipStream_t)stream;
    const int waves = sort_waves(experts);
    const int chunks = n > 0 ? (int)ceil_div(n, waves * kPerWave) : 1;
    int bits = 1;
    while ((1 << bits) < experts) bits++;
    const size_t lds = 4 * (size_t)experts + 2 * (size_t)waves * experts;
    if (chunks == 1) {
        launch(k_route_place<true>, dim3(1), dim3(64 * waves), lds, st, ids, n, experts, bits, nullptr, nullptr, offsets, order, place);
    } else {
        int *counts = (int *)workspace, *total = counts + (long long)chunks * experts;
        launch(k_route_count, dim3(chunks), dim3(64 * waves), 4 * (size_t)experts, st, ids, n, experts, counts);
        launch(k_route_prefix, dim3(experts), dim3(64), 0, st, counts, total, chunks, experts);
        launch(k_route_place<false>, dim3(chunks), dim3(64 * waves), lds, st, ids, n, experts, bits, counts, total, offsets, order, place);
    }
    return launched("route");
}

int nsparse_lm_gather_tokens(int dtype, const void *x, const int *place, long long tokens, int top, int channels, void *xs, void *stream)
{
    using namespace nsp::lm;
    clear_error();
    if (int rc = check_products(dtype, tokens, top, channels, "gather_tokens: tokens, top or channels out of range")) return rc;
    if (tokens == 0) return 0;
    if (!x || !place || !xs) return fail(NSPARSE_LM_EARG, "gather_tokens: a required pointer is NULL");
    if (((uintptr_t)x | (uintptr_t)xs) % elem_size(dtype)) return fail(NSPARSE_LM_EALIGN, "gather_tokens: x and xs begin at elements of their type");
    const int per = threads_per_token(channels, dtype);
    const dim3 grid = groups(ceil_div(tokens, 256 / per));
    hipStream_t st = (hipStream_t)stream;
#define NSP_GO(U) \
    launch(k_gather_tokens<U>, grid, dim3(256), 0, st, (const U *)x, place, (int)tokens, top, channels, per, (U *)xs)
    if (dtype == NSPARSE_LM_F32) NSP_GO(unsigned);
    else NSP_GO(unsigned short);
#undef NSP_GO
    return launched("gather_tokens");
}

int nsparse_lm_combine_tokens(int dtype, const void *y, const int *place, const float *w, long long tokens, int top, int channels, void *out,
                              void *stream)
{
    using namespace nsp::lm;
    clear_error();
    if (int rc = check_products(dtype, tokens, top, channels, "combine_tokens: tokens, top or channels out of range")) return rc;
    if (tokens == 0) return 0;
    if (!y || !place || !out) return fail(NSPARSE_LM_EARG, "combine_tokens: a required pointer is NULL");
    if (((uintptr_t)y | (uintptr_t)out) % elem_size(dtype)) return fail(NSPARSE_LM_EALIGN, "combine_tokens: y and out begin at elements of their type");
    const int per = threads_per_token(channels, dtype);
    const dim3 grid = groups(ceil_div(tokens, 256 / per));
    hipStream_t st = (hipStream_t)stream;
#define NSP_GO(T) \
    launch(k_combine_tokens<T>, grid, dim3(256), 0, st, (const T *)y, place, w, (int)tokens, top, channels, per, (T *)out)
    if (dtype == NSPARSE_LM_BF16) NSP_GO(__bf16);
    else if (dtype == NSPARSE_LM_F16) NSP_GO(_Float16);
    else NSP_GO(float);
#undef NSP_GO
    return launched("combine_tokens");
}

int nsparse_lm_combine_tokens_bwd(int dtype, const void *dout, const void *y, const int *place, const float *w, long long tokens, int top,
                                  int channels, void *dy, float *dw, void *stream)
{
    using namespace nsp::lm;
    clear_error();
    if (int rc = check_products(dtype, tokens, top, channels, "combine_tokens_bwd: tokens, top or channels out of range")) return rc;
    if (tokens == 0) return 0;
    if (!dout || !place || !dy || (dw && !y) || (w && !dw)) return fail(NSPARSE_LM_EARG, "combine_tokens_bwd: a required pointer is NULL");
    if (((uintptr_t)dout | (uintptr_t)y | (uintptr_t)dy) % elem_size(dtype))
        return fail(NSPARSE_LM_EALIGN, "combine_tokens_bwd: dout, y and dy begin at elements of their type");
    const int per = threads_per_token(channels, dtype);
    const dim3 grid = groups(ceil_div(tokens, 256 / per));
    hipStream_t st = (hipStream_t)stream;
#define NSP_GO(T)                                                                                                                 \
    launch(k_combine_tokens_bwd<T>, grid, dim3(256), 0, st, (const T *)dout, (const T *)y, place, w, (int)tokens, top, \
                       channels, per, (T *)dy, dw)
    if (dtype == NSPARSE_LM_BF16) NSP_GO(__bf16);
    else if (dtype == NSPARSE_LM_F16) NSP_GO(_Float16);
    else NSP_GO(float);
#undef NSP_GO
    return launched("combine_tokens_bwd");
}
}
