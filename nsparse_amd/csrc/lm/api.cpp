// api.cpp -- error channel and the argument checks that the attention entry points share.
#include <cfloat>
#include <cmath>
#include <cstdio>
#include <cstring>

#include "common.h"

namespace nsp {
namespace lm {

namespace {
thread_local int t_code = 0;
thread_local char t_text[256] = "";
thread_local hipError_t t_launch = hipSuccess;
}  // namespace

int fail(int code, const char *what)
{
    t_code = code;
    snprintf(t_text, sizeof(t_text), "nsparse_lm: %s", what);
    return code;
}
void clear_error()
{
    t_code = 0;
    t_text[0] = 0;
    t_launch = hipSuccess;
}
void note_launch(hipError_t e)
{
    if (e == hipSuccess) return;
    (void)hipGetLastError();  // it is returned, so it is nobody else's
    if (t_launch == hipSuccess) t_launch = e;
}
int launched(const char *what)
{
    const hipError_t e = t_launch;
    if (e == hipSuccess) return 0;
    t_code = (int)e;
    snprintf(t_text, sizeof(t_text), "nsparse_lm: %s: %s", what, hipGetErrorString(e));
    return (int)e;
}

int geometry(const nsparse_lm_attn *a, bool needs_q, bool needs_k, Geometry *g)
{
    if (!a) return fail(NSPARSE_LM_EARG, "the argument block is NULL");
    if (a->dtype != NSPARSE_LM_F32 && a->dtype != NSPARSE_LM_F16 && a->dtype != NSPARSE_LM_BF16)
        return fail(NSPARSE_LM_ETYPE, "dtype is none of F32, F16, BF16");
    if (a->heads < 1 || a->kv_heads < 1 || a->heads % a->kv_heads || a->heads / a->kv_heads > 1024)
        return fail(NSPARSE_LM_EARG, "heads must be a multiple of kv_heads, at most 1024 times as many");
    if (a->head_dim < 8 || a->head_dim > 256 || a->head_dim % 8) return fail(NSPARSE_LM_EARG, "head_dim must be a multiple of 8 up to 256");
    if (a->block < 16 || a->block > 256 || (a->block & (a->block - 1))) return fail(NSPARSE_LM_EARG, "block must be 16, 32, 64, 128 or 256");
    if (a->width < 1 || a->width > 256) return fail(NSPARSE_LM_EARG, "width must be 1 .. 256");
    // the softmax is taken in base 2: the scale times log2 e has to be a number as well
    if (!(fabsf(a->scale) * 1.4426950408889634f <= FLT_MAX)) return fail(NSPARSE_LM_EARG, "scale must be a finite number, at most 2.3e38");
    if (a->n_seq < 1) return fail(NSPARSE_LM_EARG, "n_seq must be positive");
    if (a->q_rows < 0 || a->q_rows > 0x7fffffffLL / 2 || a->k_rows < 0) return fail(NSPARSE_LM_EARG, "q_rows or k_rows out of range");
    // one workgroup index per (query row, key head, slice of 16 heads)
    if (a->q_rows * (a->kv_heads + (long long)a->heads / 16) > kMostGroups) return fail(NSPARSE_LM_EARG, "q_rows x heads out of range");
    if (a->page_size < 0 || a->page_size % a->block) return fail(NSPARSE_LM_EARG, "page_size must be a multiple of block");
    if (a->page_size > 0) {
        if (!a->k_len || !a->page_table) return fail(NSPARSE_LM_EARG, "a paged cache needs k_len and page_table");
        if (a->cu_k) return fail(NSPARSE_LM_EARG, "cu_k does not go with a paged cache");
        if (a->k_rows > 0x7fffffffLL) return fail(NSPARSE_LM_EARG, "k_rows out of range");
        if (a->table_stride < 0 || a->table_stride > 0x7fffffffLL / a->page_size) return fail(NSPARSE_LM_EARG, "table_stride out of range");
    } else {
        if (a->page_table) return fail(NSPARSE_LM_EARG, "page_table without page_size");
        if (!a->cu_k && a->k_rows % a->n_seq) return fail(NSPARSE_LM_EARG, "k_rows must divide by n_seq where cu_k is absent");
        if ((a->cu_k ? a->k_rows : a->k_rows / a->n_seq) > kMostKeys) return fail(NSPARSE_LM_EARG, "k_rows out of range");
    }
    if (!a->cu_q && a->q_rows % a->n_seq) return fail(NSPARSE_LM_EARG, "q_rows must divide by n_seq where cu_q is absent");
    const int per16 = 16 / elem_size(a->dtype);
    if (needs_q)
        for (int i = 0; i < 2; i++)
            if (a->q_stride[i] % per16 || a->q_stride[i] < 0) return fail(NSPARSE_LM_EALIGN, "q strides must be multiples of 16 bytes");
    if (needs_k)
        for (int i = a->page_size > 0 ? 0 : 1; i < 3; i++)
            if (a->k_stride[i] % per16 || a->v_stride[i] % per16 || a->k_stride[i] < 0 || a->v_stride[i] < 0)
                return fail(NSPARSE_LM_EALIGN, "k and v strides must be multiples of 16 bytes");
    Geometry &G = *g;
    memset(&G, 0, sizeof(G));
    G.n_seq = a->n_seq;
    G.heads = a->heads;
    G.kv_heads = a->kv_heads;
    G.group = a->heads / a->kv_heads;
    G.head_dim = a->head_dim;
    G.block = a->block;
    G.width = a->width;
    G.causal = a->causal != 0;
    G.page_size = a->page_size;
    G.per_page = a->page_size > 0 ? a->page_size / a->block : 1;
    G.q_rows = (int)a->q_rows;
    G.q_each = a->cu_q ? 0 : (int)(a->q_rows / a->n_seq);
    G.k_rows = a->k_rows;
    G.k_each = (a->cu_k || a->page_size > 0) ? 0 : a->k_rows / a->n_seq;
    G.blocks_each = (int)ceil_div(G.k_each, a->block);
    G.table_stride = a->table_stride;
    G.cu_q = a->cu_q;
    G.cu_k = a->cu_k;
    G.q_len = a->q_len;
    G.k_len = a->k_len;
    G.page_table = a->page_table;
    G.q_row = a->q_stride[0];
    G.q_head = a->q_stride[1];
    G.k_page = a->k_stride[0];
    G.k_row = a->k_stride[1];
    G.k_head = a->k_stride[2];
    G.v_page = a->v_stride[0];
    G.v_row = a->v_stride[1];
    G.v_head = a->v_stride[2];
    G.scale = a->scale;
    return 0;
}

}  // namespace lm
}  // namespace nsp

extern "C" {

int nsparse_lm_last_error(void) { return nsp::lm::t_code; }
const char *nsparse_lm_last_error_string(void) { return nsp::lm::t_text; }
const char *nsparse_lm_build_info(void) { return "gfx950 " NSPARSE_LM_HASH; }

long long nsparse_lm_mean_rows(const nsparse_lm_attn *a)
{
    nsp::lm::clear_error();
    nsp::lm::Geometry G;
    if (int rc = nsp::lm::geometry(a, false, false, &G)) return rc;
    if (G.page_size > 0) return G.k_rows * G.per_page;
    if (G.cu_k) return G.k_rows / G.block + G.n_seq;
    return (long long)G.blocks_each * G.n_seq;
}
}
