// yl_paged.hip -- a K/V cache in pages that many sequences share: appending
// rows to it with the position rotation on the way (yl_paged_attn.hip reads it).
// No counterpart in the reference, which holds one conversation.
#include <hip/hip_runtime.h>

#include <math.h>

#include "../../include/yallma3.h"
#include "yl_device.h"
#include "yl_internal.h"
#include "yl_paged.h"

namespace yl {

// ---------------------------------------------------------------- appending

struct AppendArgs {
    PagedArgs p;
    float* q_out; const float* q; const float* k; const float* v;
    size_t q_out_ld, q_ld, k_ld, v_ld;
    int pairs;                       // YL_ROPE_*
    const float* cos_t; const float* sin_t;
    int64_t rope_rows;
};

// One workgroup per row; a thread per pair of a query or key head, then one
// per pair of value elements.
template <typename C>
__global__ __launch_bounds__(256) void k_paged_append(AppendArgs a) {
    const int row = blockIdx.x, hd = a.p.hd, half = hd / 2, tid = threadIdx.x;
    const int s = paged_seq_of_row(a.p, row);
    if (s < 0) return;
    int first, end;
    paged_rows(a.p, s, &first, &end);
    if (row < first || row >= end) return;
    const int64_t pos = paged_row_pos(a.p.kv_len[s], end, row);
    if (pos < 0 || (a.pairs != YL_ROPE_NONE && pos >= a.rope_rows)) return;
    int page = -1, slot = 0;
    const bool keep = pos >= a.p.prefix_len && paged_place(a.p, s, pos, &page, &slot);
    const int nq = a.q ? a.p.n_heads * half : 0, nk = a.p.n_kv * half;
    for (int i = tid; i < nq + nk; i += 256) {
        const bool is_q = i < nq;
        const int j = is_q ? i : i - nq, head = j / half, e = j % half;
        const int lo = a.pairs == YL_ROPE_HALF ? e : 2 * e, hi = a.pairs == YL_ROPE_HALF ? e + half : 2 * e + 1;
        const float* x = (is_q ? a.q + (size_t)row * a.q_ld : a.k + (size_t)row * a.k_ld) + (size_t)head * hd;
        float x0 = x[lo], x1 = x[hi];
        if (a.pairs != YL_ROPE_NONE) {
            const float c = a.cos_t[(size_t)pos * half + e], sn = a.sin_t[(size_t)pos * half + e];
            const float r0 = fmul(x0, c) - fmul(x1, sn), r1 = fadd(fmul(x0, sn), fmul(x1, c));
            x0 = r0;
            x1 = r1;
        }
        if (is_q) {
            float* o = a.q_out + (size_t)row * a.q_out_ld + (size_t)head * hd;
            o[lo] = x0;
            o[hi] = x1;
        } else if (keep) {
            C* o = static_cast<C*>(a.p.keys) + paged_offset(a.p, page, head, slot);
            o[lo] = (C)x0;
            o[hi] = (C)x1;
        }
    }
    if (keep)
        for (int i = tid; i < a.p.n_kv * hd; i += 256)
            static_cast<C*>(a.p.values)[paged_offset(a.p, page, i / hd, slot) + i % hd] = (C)a.v[(size_t)row * a.v_ld + i];
}

// ------------------------------------------------------------- host entries

namespace {

yl_status refuse(const char* what, yl_status st = YL_ERR_ARG) {
    set_error(what);
    return st;
}

}  // namespace

yl_status paged_args(const yl_paged_cache* c, const yl_paged_batch* b, uint32_t n_heads, PagedArgs* a) {
    if (!c || !b) return refuse("paged: no cache or no batch");
    if (c->dtype != YL_T_F32 && c->dtype != YL_T_F16 && c->dtype != YL_T_BF16)
        return refuse("paged: the cache's type is f32, f16 or bf16", YL_ERR_FORMAT);
    if (c->head_size != 32 && c->head_size != 64 && c->head_size != 128) return refuse("paged: head size 32, 64 or 128");
    if (c->page_size != 16 && c->page_size != 32 && c->page_size != 64 && c->page_size != 128 && c->page_size != 256)
        return refuse("paged: page size 16, 32, 64, 128 or 256");
    if (!c->n_pages || (uint64_t)c->n_pages * c->page_size >= (1ull << 31)) return refuse("paged: n_pages * page_size from 1 page to below 2^31");
    if (!c->n_kv_heads || !n_heads || n_heads % c->n_kv_heads || n_heads > 1024)
        return refuse("paged: n_heads (at most 1024) is a multiple of n_kv_heads");
    if (!c->keys || !c->values || ((uintptr_t)c->keys | (uintptr_t)c->values) % 16)
        return refuse("paged: keys and values have to be there, 16-byte aligned");
    if ((uint64_t)b->n_rows * n_heads >= (1ull << 24) || (uint64_t)b->n_seqs * n_heads >= (1ull << 22) ||
        (uint64_t)b->prefix_len + (uint64_t)b->max_pages * c->page_size >= (1ull << 30))
        return refuse("paged: n_rows * n_heads below 2^24, n_seqs * n_heads below 2^22, a sequence's capacity below 2^30", YL_ERR_RANGE);
    if (!b->row_start && b->n_rows != b->n_seqs) return refuse("paged: without row_start there is one row per sequence");
    if (b->n_rows && b->n_seqs && (!b->kv_len || (b->max_pages && !b->page_table)))
        return refuse("paged: kv_len and page_table have to be there");
    if (b->prefix_len && !b->prefix_pages) return refuse("paged: a prefix needs prefix_pages");
    *a = PagedArgs{c->keys, c->values, (int)c->n_pages, __builtin_ctz(c->page_size), (int)c->n_kv_heads, (int)c->head_size,
                   (int)b->n_seqs, (int)b->n_rows, (int)b->max_pages, b->page_table, b->kv_len, b->row_start,
                   (int)b->prefix_len, b->prefix_pages, (int)n_heads};
    return YL_OK;
}

namespace {

yl_status launched(const char* what) {
    const hipError_t e = hipGetLastError();
    if (e == hipSuccess) return YL_OK;
    set_error(std::string(what) + ": " + hipGetErrorString(e));
    return YL_ERR_HIP;
}

}  // namespace
}  // namespace yl

using namespace yl;

extern "C" {

yl_status yl_paged_append(const yl_paged_cache* cache, const yl_paged_batch* batch, uint32_t n_heads, float* q_out,
                          size_t q_out_ld, const float* q, size_t q_ld, const float* k, size_t k_ld, const float* v,
                          size_t v_ld, int32_t pairs, const float* cos_t, const float* sin_t, uint32_t rope_rows,
                          void* stream) {
    AppendArgs a{};
    const yl_status st = paged_args(cache, batch, n_heads, &a.p);
    if (st != YL_OK) return st;
    const size_t att = (size_t)n_heads * cache->head_size, kv = (size_t)cache->n_kv_heads * cache->head_size;
    if (pairs != YL_ROPE_NONE && pairs != YL_ROPE_ADJACENT && pairs != YL_ROPE_HALF)
        return refuse("paged_append: pairs adjacent, half or none");
    if (pairs != YL_ROPE_NONE && (!cos_t || !sin_t)) return refuse("paged_append: a rotation needs cos_t and sin_t");
    if (!batch->n_rows || !batch->n_seqs) return YL_OK;
    if (!k || !v || !q != !q_out) return refuse("paged_append: k and v, and q with q_out or neither");
    if (k_ld < kv || v_ld < kv || (q && (q_ld < att || q_out_ld < att))) return refuse("paged_append: rows further apart than they are long");
    if (q == q_out && q_ld != q_out_ld) return refuse("paged_append: in place, q_ld and q_out_ld are the same");
    a.q_out = q_out; a.q = q; a.k = k; a.v = v;
    a.q_out_ld = q_out_ld; a.q_ld = q_ld; a.k_ld = k_ld; a.v_ld = v_ld;
    a.pairs = pairs; a.cos_t = cos_t; a.sin_t = sin_t; a.rope_rows = rope_rows;
    auto kern = cache->dtype == YL_T_F32 ? k_paged_append<float> : cache->dtype == YL_T_F16 ? k_paged_append<_Float16> : k_paged_append<__bf16>;
    hipLaunchKernelGGL(kern, dim3(batch->n_rows), dim3(256), 0, (hipStream_t)stream, a);
    return launched("paged_append launch");
}

}  // extern "C"
