// yl_paged.hip -- a K/V cache in pages that many sequences share: appending
// rows to it with the position rotation on the way (yl_paged_attn.hip reads it),
// and bringing rows back out of it.
// No counterpart in the reference, which holds one conversation.
#include <hip/hip_runtime.h>

#include <math.h>

#include <type_traits>

#include "../../include/yallma3.h"
#include "yl_device.h"
#include "yl_internal.h"
#include "yl_mx.h"
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

typedef float f4u __attribute__((ext_vector_type(4), aligned(4)));   // activations: any float address
typedef float f2u __attribute__((ext_vector_type(2), aligned(4)));

// Four neighbouring elements rounded to the cache's type, once, to nearest.
template <typename C>
__device__ __forceinline__ void store4(C* o, const f4u& x) {
    typedef C c4 __attribute__((ext_vector_type(4)));
    *reinterpret_cast<c4*>(o) = __builtin_convertvector((vf4{x[0], x[1], x[2], x[3]}), c4);
}

template <typename C> constexpr bool kMx = std::is_same<C, Mx4>::value;

__device__ __forceinline__ uint32_t amax4(const f4u& x) {
    uint32_t m = 0;
#pragma unroll
    for (int k = 0; k < 4; k++) m = max(m, __float_as_uint(x[k]) & 0x7fffffffu);
    return m;
}

// Four neighbouring elements from `e` on of a slot's head in MXFP4, whose block's largest has the bits `amax`.
__device__ __forceinline__ void store_mx(const PagedArgs& p, void* pool, int page, int head, int slot, int e, const f4u& x, uint32_t amax) {
    const uint32_t scale = mx_scale(amax);
    char* base = static_cast<char*>(pool);
    const uint32_t codes = mx_codes(x[0], x[1], x[2], x[3], mx_unit(scale));
    *reinterpret_cast<uint16_t*>(base + paged_mx_codes(p, page, head, slot) + e / 2) = (uint16_t)codes;
    if (e % 32 == 0) base[paged_mx_scales(p, page, head, slot) + e / 32] = (char)scale;
}

// The sequence of a row by a whole wavefront, 64 starts per step (as paged_seq_of_row).
__device__ __forceinline__ int seq_of_row(const PagedArgs& a, int row) {
    if (!a.row_start) return row < a.n_seqs ? row : -1;
    const int lane = threadIdx.x & 63;
    int lo = 0, n = a.n_seqs;                 // the last start not above the row is one of lo .. lo + n - 1
    while (n > 1) {
        const int step = (n + 63) >> 6;
        const bool ok = lane * step < n && a.row_start[lo + lane * step] <= (uint32_t)row;
        const int c = max(1, (int)__builtin_popcountll(__ballot(ok))) - 1;
        lo += c * step;
        n = min(step, n - c * step);
    }
    lo = __builtin_amdgcn_readfirstlane(lo);
    return a.row_start[lo] <= (uint32_t)row && (uint32_t)row < a.row_start[lo + 1] ? lo : -1;
}

// One workgroup per row; a thread takes 4 neighbouring elements (of a half
// rotation, 4 pairs) at a time.  Bound by memory: 16-byte loads, several in
// flight per thread: 9751 rows of 32 + 8 + 8 heads of 128, f16, 84 us, 5.3 TB/s
// (a pair per thread and pass: 112 us); a decoded row 3 us, the launch.  Into MXFP4
// pages a block's 32 elements stand in 8 neighbouring lanes, whose largest three
// lane exchanges find; 2 bytes of codes per lane: 9751 rows of 32 + 8 + 8 heads of 64
// 34 us, 6.0 TB/s (so many rows are stores that the writes of q bound it).
template <typename C, int PAIRS>
__global__ __launch_bounds__(256) void k_paged_append(AppendArgs a) {
    const int row = blockIdx.x, hd = a.p.hd, half = hd / 2, tid = threadIdx.x;
    const int s = seq_of_row(a.p, row);
    if (s < 0) return;
    int first, end;
    paged_rows(a.p, s, &first, &end);
    if (row < first || row >= end) return;
    const int64_t pos = paged_row_pos(a.p.kv_len[s], end, row);
    if (pos < 0 || (PAIRS != YL_ROPE_NONE && pos >= a.rope_rows)) return;
    int page = -1, slot = 0;
    const bool keep = pos >= a.p.prefix_len && paged_place(a.p, s, pos, &page, &slot);
    const float* ct = a.cos_t + (size_t)pos * half;
    const float* st = a.sin_t + (size_t)pos * half;
    // element offset of (head, element) in a page
    const auto at = [&](int head, int e) { return paged_offset(a.p, page, head, slot) + e; };
    const int shift = 31 - __builtin_clz(hd);             // (hd is a power of two)
    const float* qr = a.q + (size_t)row * a.q_ld;
    const float* kr = a.k + (size_t)row * a.k_ld;
    const float* vr = a.v + (size_t)row * a.v_ld;
    float* qo = a.q_out + (size_t)row * a.q_out_ld;
    const int nq = a.q ? a.p.n_heads * hd : 0, nk = keep ? a.p.n_kv * hd : 0;
    if constexpr (PAIRS == YL_ROPE_HALF) {
        const int uq = nq / 8, uk = nk / 8;               // units of 4 pairs
#pragma unroll kMx<C> ? 1 : 2
        for (int i = tid; i < uq + uk; i += 256) {
            const bool is_q = i < uq;
            const int j = is_q ? i : i - uq, head = j >> (shift - 3), e = 4 * (j & (hd / 8 - 1));
            const float* x = (is_q ? qr : kr) + (size_t)head * hd + e;
            const f4u x0 = *reinterpret_cast<const f4u*>(x), x1 = *reinterpret_cast<const f4u*>(x + half);
            const f4u c = *reinterpret_cast<const f4u*>(ct + e), sn = *reinterpret_cast<const f4u*>(st + e);
            f4u r0, r1;
#pragma unroll
            for (int k = 0; k < 4; k++) {
                r0[k] = fmul(x0[k], c[k]) - fmul(x1[k], sn[k]);
                r1[k] = fadd(fmul(x0[k], sn[k]), fmul(x1[k], c[k]));
            }
            if (is_q) {
                *reinterpret_cast<f4u*>(qo + (size_t)head * hd + e) = r0;
                *reinterpret_cast<f4u*>(qo + (size_t)head * hd + e + half) = r1;
            } else if constexpr (kMx<C>) {
                // (a head's lanes stand together: half / 4 of them, 8 to a block of one half, at hd 32 all 4 of both)
                const uint32_t m0 = amax4(r0), m1 = amax4(r1);
                const uint32_t b0 = hd == 32 ? mx_group_max<4>(max(m0, m1)) : mx_group_max<8>(m0);
                const uint32_t b1 = hd == 32 ? b0 : mx_group_max<8>(m1);
                store_mx(a.p, a.p.keys, page, head, slot, e, r0, b0);
                store_mx(a.p, a.p.keys, page, head, slot, e + half, r1, b1);
            } else {
                C* o = static_cast<C*>(a.p.keys) + at(head, e);
                store4(o, r0);
                store4(o + half, r1);
            }
        }
    } else {
        const int uq = nq / 4, uk = nk / 4;
#pragma unroll kMx<C> ? 1 : 4
        for (int i = tid; i < uq + uk; i += 256) {
            const bool is_q = i < uq;
            const int j = is_q ? i : i - uq, head = j >> (shift - 2), e = 4 * (j & (hd / 4 - 1));
            f4u x = *reinterpret_cast<const f4u*>((is_q ? qr : kr) + 4 * (size_t)j);
            if constexpr (PAIRS == YL_ROPE_ADJACENT) {
                const f2u c = *reinterpret_cast<const f2u*>(ct + e / 2), sn = *reinterpret_cast<const f2u*>(st + e / 2);
                f4u r;
#pragma unroll
                for (int k = 0; k < 2; k++) {
                    r[2 * k] = fmul(x[2 * k], c[k]) - fmul(x[2 * k + 1], sn[k]);
                    r[2 * k + 1] = fadd(fmul(x[2 * k], sn[k]), fmul(x[2 * k + 1], c[k]));
                }
                x = r;
            }
            if (is_q) *reinterpret_cast<f4u*>(qo + 4 * (size_t)j) = x;
            else if constexpr (kMx<C>) store_mx(a.p, a.p.keys, page, head, slot, e, x, mx_group_max<8>(amax4(x)));
            else store4(static_cast<C*>(a.p.keys) + at(head, e), x);
        }
    }
#pragma unroll kMx<C> ? 1 : 2
    for (int j = tid; j < nk / 4; j += 256) {
        const f4u x = *reinterpret_cast<const f4u*>(vr + 4 * (size_t)j);
        const int head = j >> (shift - 2), e = 4 * (j & (hd / 4 - 1));
        if constexpr (kMx<C>) store_mx(a.p, a.p.values, page, head, slot, e, x, mx_group_max<8>(amax4(x)));
        else store4(static_cast<C*>(a.p.values) + at(head, e), x);
    }
}

// ----------------------------------------------------------------- gathering

struct GatherArgs {
    PagedArgs p;
    float* k; float* v;
    size_t k_ld, v_ld;
};

// Four neighbouring elements of a slot's head, widened.
template <typename C>
__device__ __forceinline__ f4u load4(const PagedArgs& p, const void* pool, int page, int head, int slot, int e) {
    if constexpr (kMx<C>) {
        const char* base = static_cast<const char*>(pool);
        const uint32_t codes = *reinterpret_cast<const uint16_t*>(base + paged_mx_codes(p, page, head, slot) + e / 2);
        const float unit = mx_unit((uint8_t)base[paged_mx_scales(p, page, head, slot) + e / 32]);
        const uint32_t lo = mx_pair<0>(codes, unit), hi = mx_pair<1>(codes, unit);
        return f4u{__uint_as_float(lo << 16), __uint_as_float(lo & 0xffff0000u), __uint_as_float(hi << 16), __uint_as_float(hi & 0xffff0000u)};
    } else {
        typedef C c4 __attribute__((ext_vector_type(4)));
        const c4 x = *reinterpret_cast<const c4*>(static_cast<const C*>(pool) + paged_offset(p, page, head, slot) + e);
        return f4u{(float)x[0], (float)x[1], (float)x[2], (float)x[3]};
    }
}

// One workgroup per row, as k_paged_append.  Bound by memory, nearly all of it what
// is written: 9751 rows of 8 heads of 64, keys and values, out of MXFP4 pages 15 us,
// 6.1 TB/s; 64 rows 3 us, the launch.  (Stores that L2 does not keep, and a longer unrolling,
// changed it by less than 1%.)
template <typename C>
__global__ __launch_bounds__(256) void k_paged_gather(GatherArgs a) {
    const int row = blockIdx.x, hd = a.p.hd, tid = threadIdx.x;
    const int s = seq_of_row(a.p, row);
    if (s < 0) return;
    int first, end;
    paged_rows(a.p, s, &first, &end);
    if (row < first || row >= end) return;
    const int64_t pos = paged_row_pos(a.p.kv_len[s], end, row);
    int page = -1, slot = 0;
    if (pos < 0 || !paged_place(a.p, s, pos, &page, &slot)) return;
    const int shift = 31 - __builtin_clz(hd), n = a.p.n_kv * hd / 4;
#pragma unroll 2
    for (int i = tid; i < 2 * n; i += 256) {
        const bool key = i < n;
        const int j = key ? i : i - n;
        float* out = key ? a.k : a.v;
        if (!out) continue;
        const f4u x = load4<C>(a.p, key ? a.p.keys : a.p.values, page, j >> (shift - 2), slot, 4 * (j & (hd / 4 - 1)));
        *reinterpret_cast<f4u*>(out + (size_t)row * (key ? a.k_ld : a.v_ld) + 4 * (size_t)j) = x;
    }
}

// ------------------------------------------------------------- host entries

namespace {

yl_status refuse(const char* what, yl_status st = YL_ERR_ARG) {
    set_error(what);
    return st;
}

}  // namespace

yl_status paged_cache_ok(const yl_paged_cache* c) {
    if (c->dtype != YL_T_F32 && c->dtype != YL_T_F16 && c->dtype != YL_T_BF16 && c->dtype != YL_T_MXFP4)
        return refuse("paged: the cache's type is f32, f16, bf16 or MXFP4", YL_ERR_FORMAT);
    if (c->head_size != 32 && c->head_size != 64 && c->head_size != 128) return refuse("paged: head size 32, 64 or 128");
    if (c->page_size != 16 && c->page_size != 32 && c->page_size != 64 && c->page_size != 128 && c->page_size != 256)
        return refuse("paged: page size 16, 32, 64, 128 or 256");
    if (!c->n_pages || (uint64_t)c->n_pages * c->page_size >= (1ull << 31)) return refuse("paged: n_pages * page_size from 1 page to below 2^31");
    if (!c->keys || !c->values || ((uintptr_t)c->keys | (uintptr_t)c->values) % 16)
        return refuse("paged: keys and values have to be there, 16-byte aligned");
    if (!c->n_kv_heads || c->n_kv_heads > 1024) return refuse("paged: n_kv_heads from 1 to 1024");
    return YL_OK;
}

yl_status paged_args(const yl_paged_cache* c, const yl_paged_batch* b, uint32_t n_heads, PagedArgs* a) {
    if (!c || !b) return refuse("paged: no cache or no batch");
    const yl_status st = paged_cache_ok(c);
    if (st != YL_OK) return st;
    if (!n_heads || n_heads % c->n_kv_heads || n_heads > 1024) return refuse("paged: n_heads (at most 1024) is a multiple of n_kv_heads");
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

template <typename C>
void launch_append(const AppendArgs& a, hipStream_t s) {
    auto k = a.pairs == YL_ROPE_HALF ? k_paged_append<C, YL_ROPE_HALF> : a.pairs == YL_ROPE_ADJACENT ? k_paged_append<C, YL_ROPE_ADJACENT>
                                                                                                  : k_paged_append<C, YL_ROPE_NONE>;
    hipLaunchKernelGGL(k, dim3(a.p.n_rows), dim3(256), 0, s, a);
}

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
    const hipStream_t strm = (hipStream_t)stream;
    if (cache->dtype == YL_T_F32) launch_append<float>(a, strm);
    else if (cache->dtype == YL_T_F16) launch_append<_Float16>(a, strm);
    else if (cache->dtype == YL_T_BF16) launch_append<__bf16>(a, strm);
    else launch_append<Mx4>(a, strm);
    return launched("paged_append launch");
}

yl_status yl_paged_gather(const yl_paged_cache* cache, const yl_paged_batch* batch, float* k, size_t k_ld, float* v, size_t v_ld,
                          void* stream) {
    GatherArgs a{};
    const yl_status st = paged_args(cache, batch, cache ? cache->n_kv_heads : 0, &a.p);
    if (st != YL_OK) return st;
    if (!k && !v) return refuse("paged_gather: k or v, or both");
    const size_t kv = (size_t)cache->n_kv_heads * cache->head_size;
    if ((k && k_ld < kv) || (v && v_ld < kv)) return refuse("paged_gather: rows further apart than they are long");
    if (!batch->n_rows || !batch->n_seqs) return YL_OK;
    a.k = k; a.v = v; a.k_ld = k_ld; a.v_ld = v_ld;
    const hipStream_t strm = (hipStream_t)stream;
    auto kernel = cache->dtype == YL_T_F32 ? k_paged_gather<float> : cache->dtype == YL_T_F16 ? k_paged_gather<_Float16>
                  : cache->dtype == YL_T_BF16 ? k_paged_gather<__bf16> : k_paged_gather<Mx4>;
    hipLaunchKernelGGL(kernel, dim3(a.p.n_rows), dim3(256), 0, strm, a);
    return launched("paged_gather launch");
}

}  // extern "C"
