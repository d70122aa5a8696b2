// yl_paged_attn.hip -- causal attention over a paged cache (yl_paged_attention).
//
// Per kv head, the rows that attend to the same pages are stacked: (token,
// query head of the group) with the heads fastest.  A tile is 16 such rows, the
// N side of the matrix instructions:
//   S^T [positions][rows] = K Q^T,   O^T [dims][rows] = V^T P^T.
// With the rows on N, a lane (c = lane % 16, g = lane / 16) holds in both
// results values of row c only, so maxima, sums and rescalings are per lane,
// and S^T's registers are P^T's operand as they are: of a 16-position tile lane
// group g holds positions 4g .. 4g + 3, and the order of positions inside a
// product is free as long as V's operand has the same one.  V^T's operand
// wants one dimension of 8 positions per lane while rows are stored dimension
// by dimension: a lane loads HD / 16 neighbouring dimensions of its 8 positions
// and picks each dimension's halves with v_perm, no lane exchange.
//
// Precision: the products run on f16 / bf16 matrix instructions with f32 sums
// while q and the weights are f32, so these are cut into parts that add up to
// them: two f16 (22 bits; q scaled per row by a power of two, the weights by
// 2^kBias, so that the second part keeps its bits) or three bf16 (24 bits).  f32
// caches take the f32 matrix instructions.
//
// Softmax: running maximum and sum per row in base 2 (one pass over the keys).
// The maximum is only raised when a score passes it by more than 2^kSlack.
#include <hip/hip_runtime.h>

#include <math.h>

#include <algorithm>

#include "../../include/yallma3.h"
#include "yl_device.h"
#include "yl_internal.h"
#include "yl_paged.h"

namespace yl {

namespace {

typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));
typedef uint32_t u2 __attribute__((ext_vector_type(2)));
typedef float f4u __attribute__((ext_vector_type(4), aligned(4)));   // activations: any float address

constexpr float kSlack = 8.0f;      // a score may pass the running maximum by this power of two

// What depends on the cache's type.
template <typename C> struct Type;
template <> struct Type<_Float16> {
    static constexpr int kParts = 2, kTiles = 2;   // parts of an f32 value; 16-position tiles of one step
    // weights are held times 2^6: at most 2^14 with the slack, and a weight's
    // second part keeps its bits down to 2^-30
    static constexpr float kBias = 6.0f;
    static __device__ __forceinline__ vf4 mul(u4 a, u4 b, vf4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c, 0, 0, 0);
    }
    // two values -> their parts, packed
    static __device__ __forceinline__ void cut(float a, float b, uint32_t part[2]) {
        const h2 hi = __builtin_convertvector(vf2{a, b}, h2);
        const h2 lo = __builtin_convertvector((vf2{a - (float)hi[0], b - (float)hi[1]}), h2);
        part[0] = __builtin_bit_cast(uint32_t, hi);
        part[1] = __builtin_bit_cast(uint32_t, lo);
    }
    // the power of two that brings a row of q to [2^9, 2^10)
    static __device__ __forceinline__ int exponent(float amax) {
        return amax > 0.0f && amax < INFINITY ? min(9 - __builtin_amdgcn_frexp_expf(amax), 110) : 0;
    }
    static __device__ __forceinline__ bool finite(uint32_t two) { return (two & 0x7c00u) != 0x7c00u && (two & 0x7c000000u) != 0x7c000000u; }
    static __device__ __forceinline__ float widen(uint32_t two, int half) { return f16_to_f32((uint16_t)(half ? two >> 16 : two)); }
};
template <> struct Type<__bf16> {
    static constexpr int kParts = 3, kTiles = 2;
    static constexpr float kBias = 0.0f;
    static __device__ __forceinline__ vf4 mul(u4 a, u4 b, vf4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, a), __builtin_bit_cast(b8, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ uint32_t high(float a, float b) {   // cut off, not rounded: the next part takes the rest
        return __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302);
    }
    static __device__ __forceinline__ void cut(float a, float b, uint32_t part[3]) {
#pragma unroll
        for (int p = 0; p < 3; p++) {
            part[p] = high(a, b);
            a -= __uint_as_float(part[p] << 16);
            b -= __uint_as_float(part[p] & 0xffff0000u);
        }
    }
    static __device__ __forceinline__ int exponent(float) { return 0; }
    static __device__ __forceinline__ bool finite(uint32_t two) { return (two & 0x7f80u) != 0x7f80u && (two & 0x7f800000u) != 0x7f800000u; }
    static __device__ __forceinline__ float widen(uint32_t two, int half) { return __uint_as_float(half ? two & 0xffff0000u : two << 16); }
};
template <> struct Type<float> {
    static constexpr int kParts = 1, kTiles = 1;
    static constexpr float kBias = 0.0f;
    static __device__ __forceinline__ int exponent(float) { return 0; }
};

// Words a vector of N consecutive cache elements takes.
template <int W> struct Words { uint32_t w[W]; };

template <int W>
__device__ __forceinline__ Words<W> load_words(const void* p) {
    Words<W> r;
    if constexpr (W % 4 == 0) {
#pragma unroll
        for (int i = 0; i < W / 4; i++) {
            const u4 v = reinterpret_cast<const u4*>(p)[i];
#pragma unroll
            for (int k = 0; k < 4; k++) r.w[4 * i + k] = v[k];
        }
    } else if constexpr (W == 2) {
        const u2 v = *reinterpret_cast<const u2*>(p);
        r.w[0] = v[0]; r.w[1] = v[1];
    } else {
        static_assert(W == 1, "1, 2 or a multiple of 4 words");
        r.w[0] = *reinterpret_cast<const uint32_t*>(p);
    }
    return r;
}

__device__ __forceinline__ float group_max16(float v) {   // over the lanes of one row: l, l ^ 16, l ^ 32, l ^ 48
    v = fmaxf(v, __shfl_xor(v, 16, 64));
    return fmaxf(v, __shfl_xor(v, 32, 64));
}
__device__ __forceinline__ float group_sum16(float v) {
    v += __shfl_xor(v, 16, 64);
    return v + __shfl_xor(v, 32, 64);
}

}  // namespace

// What one call's kernels share.
struct PagedAttn {
    PagedArgs p;
    float* out; const float* q;
    size_t out_ld, q_ld;
    float scale_log2;                // attn_scale * log2(e)
    int group;                       // query heads per kv head
    int parts, part0;                // partial results per row and head; the first of this launch's
    int chunk;                       // positions of a split at least
    int splits;
    float* po;                       // [n_rows * n_heads][parts][hd], unnormalised
    float2* pml;                     // [n_rows * n_heads][parts]: maximum (base 2), sum; maximum -inf: nothing there
};

// A tile of the stacked rows that attend to the same pages.
struct RowSet {
    const int32_t* pages; int entries;   // entry of position i: pages[i >> page_shift], i < entries << page_shift
    int first, rows;                     // rows of the batch; stacked row i is row first + i / group
    int seq;                             // sequence, or -1: the whole batch over the prefix
};

// The tile of slot `slot`: sequence s takes slots from floor(row_start[s] *
// group / 16) + s on, of which it uses one per 16 stacked rows: a sequence's
// slots always suffice, and are found by a search over row_start alone (64
// starts per step, one per lane).  False: a slot that nothing uses.
__device__ __forceinline__ bool tile_of_slot(const PagedAttn& a, int slot, int rows_log2, RowSet* set, int* tile) {
    const PagedArgs& p = a.p;
    set->entries = p.max_pages;
    if (!p.row_start) {
        const int per = (a.group + (1 << rows_log2) - 1) >> rows_log2;
        set->seq = slot / per;
        *tile = slot - set->seq * per;
        set->first = set->seq;
        set->rows = 1;
    } else {
        const int lane = threadIdx.x & 63;
        const auto base = [&](int s) {
            const uint32_t st = p.row_start[s];
            return (int)(((int64_t)(st < (uint32_t)p.n_rows ? (int)st : p.n_rows) * a.group) >> rows_log2) + s;
        };
        int lo = 0, n = p.n_seqs;
        while (n > 1) {
            const int step = (n + 63) >> 6;
            const bool ok = lane * step < n && base(lo + lane * step) <= slot;
            const int c = max(1, (int)__builtin_popcountll(__ballot(ok))) - 1;
            lo += c * step;
            n = min(step, n - c * step);
        }
        lo = __builtin_amdgcn_readfirstlane(lo);
        set->seq = lo;
        *tile = slot - base(lo);
        int end;
        paged_rows(p, lo, &set->first, &end);
        set->rows = end - set->first;
    }
    set->pages = p.table + (size_t)set->seq * p.max_pages;
    return *tile >= 0 && ((int64_t)*tile << rows_log2) < (int64_t)set->rows * a.group;
}

// How many positions of the set's pages the row may attend to.
__device__ __forceinline__ int limit_of_row(const PagedAttn& a, const RowSet& set, int row) {
    int s = set.seq, first, end;
    if (s < 0) {                          // over the prefix: the row's own sequence
        s = paged_seq_of_row(a.p, row);
        if (s < 0) return 0;
        paged_rows(a.p, s, &first, &end);
        if (row < first || row >= end) return 0;
    } else {
        end = set.first + set.rows;
    }
    const int lim = paged_limit(a.p, paged_row_pos(a.p.kv_len[s], end, row));
    return set.seq < 0 ? min(lim, a.p.prefix_len) : max(lim - a.p.prefix_len, 0);
}

constexpr int kRowTile = 16;

// One tile of 16 stacked rows over one split of the positions, the positions
// dealt to four wavefronts in steps of 16 kTiles.  K and V go from memory to
// registers in the operands' order; the next step's keys are loaded while
// this one is computed.  Bound by memory: with few rows per kv head a byte of
// the cache meets about as many operations as the matrix cores need.
template <typename C, int HD>
__global__ __launch_bounds__(256, 2) void k_paged_attn_rows(PagedAttn a, int prefix) {
    using T = Type<C>;
    constexpr int NT = T::kTiles, NP = T::kParts, STEP = 16 * NT;
    constexpr bool F32 = sizeof(C) == 4;
    constexpr int NJ = HD / 16;                       // dimensions per lane of V, tiles of O^T
    constexpr int NK = F32 ? HD / 16 : HD / 32;       // 16-byte loads of a key per lane
    constexpr int VW = NJ * (int)sizeof(C) / 4;       // words of a V row per lane
    constexpr int LD = HD + 4;
    __shared__ __align__(16) float so[4][kRowTile][LD];
    __shared__ float sm[4][kRowTile], sl[4][kRowTile];

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int c = lane & 15, g = lane >> 4;
    const int kvh = blockIdx.x % a.p.n_kv, slot = blockIdx.x / a.p.n_kv, split = blockIdx.y;
    RowSet set;
    int tile;
    if (prefix) {
        set = RowSet{a.p.prefix_pages, (a.p.prefix_len + (1 << a.p.page_shift) - 1) >> a.p.page_shift, 0, a.p.n_rows, -1};
        tile = slot;
    } else if (!tile_of_slot(a, slot, 4, &set, &tile)) {
        return;
    }

    // this lane's row: stacked row tile * 16 + c
    const int stacked = tile * kRowTile + c;
    const bool live = stacked < set.rows * a.group;
    const int row = set.first + (live ? stacked / a.group : 0), head = kvh * a.group + (live ? stacked % a.group : 0);
    int lim = live ? limit_of_row(a, set, row) : 0;
    int most = lim;                                   // the tile's longest row
    for (int o = 1; o < 16; o <<= 1) most = max(most, __shfl_xor(most, o, 64));
    most = __builtin_amdgcn_readfirstlane(min((int64_t)most, (int64_t)set.entries << a.p.page_shift));
    const bool whole = a.splits == 1 && a.parts == 1;   // this workgroup sees all there is
    int lo = 0, hi = most;
    if (a.splits > 1) {
        const int even = (most + a.splits - 1) / a.splits;
        const int chunk = max(a.chunk, (even + 127) & ~127);
        lo = (int)min((int64_t)split * chunk, (int64_t)most);
        hi = min(lo + chunk, most);
    }
    const size_t part_at = ((size_t)row * a.p.n_heads + head) * a.parts + a.part0 + split;
    if (lo >= hi && !whole) {
        if (live && wave == 0 && g == 0) a.pml[part_at] = make_float2(-INFINITY, 0.0f);
        return;
    }
    if (!live) lim = most;                            // (spare rows follow the longest, so that they need no masks)
    int least = lim;
    for (int o = 1; o < 16; o <<= 1) least = min(least, __shfl_xor(least, o, 64));
    least = __builtin_amdgcn_readfirstlane(least);

    // q of the lane's row, cut into parts, in the order of the keys' loads
    u4 qf[NP][NK];
    float unscale = a.scale_log2;
    {
        const float* qr = a.q + (size_t)row * a.q_ld + (size_t)head * HD + (F32 ? 4 * g : 8 * g);
        f4u v[NK][F32 ? 1 : 2];
        float amax = 0.0f;
#pragma unroll
        for (int k = 0; k < NK; k++)
#pragma unroll
            for (int e = 0; e < (F32 ? 1 : 2); e++) {
                v[k][e] = *reinterpret_cast<const f4u*>(qr + k * (F32 ? 16 : 32) + 4 * e);
                if (!live) v[k][e] = f4u{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int i = 0; i < 4; i++) amax = fmaxf(amax, fabsf(v[k][e][i]));
            }
        if constexpr (F32) {
#pragma unroll
            for (int k = 0; k < NK; k++) qf[0][k] = __builtin_bit_cast(u4, v[k][0]);
        } else {
            const int ex = T::exponent(group_max16(amax));
            if (ex) unscale = __builtin_amdgcn_ldexpf(a.scale_log2, -ex);
#pragma unroll
            for (int k = 0; k < NK; k++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    uint32_t part[NP];
                    T::cut(__builtin_amdgcn_ldexpf(v[k][i >> 1][2 * (i & 1)], ex), __builtin_amdgcn_ldexpf(v[k][i >> 1][2 * (i & 1) + 1], ex), part);
#pragma unroll
                    for (int p = 0; p < NP; p++) qf[p][k][i] = part[p];
                }
        }
    }

    vf4 acc[NJ];
#pragma unroll
    for (int j = 0; j < NJ; j++) acc[j] = vf4{0.0f, 0.0f, 0.0f, 0.0f};
    float m = -INFINITY, l = 0.0f;                    // l: this lane's positions only

    const C* keys = static_cast<const C*>(a.p.keys);
    const C* values = static_cast<const C*>(a.p.values);
    const int slots = (1 << a.p.page_shift) - 1;
    const int steps = (hi - lo + STEP - 1) / STEP;
    // Pages of this wavefront's next 64 tiles, one per lane (-1: none, or past hi).
    const auto pages_from = [&](int step) {
        const int at = lo + STEP * (step + 4 * (lane / NT)) + 16 * (lane % NT);
        return at < hi ? paged_page(set.pages[at >> a.p.page_shift], a.p.n_pages) : -1;
    };
    int page_reg = pages_from(wave), page_n = 0;
    const auto tile_page = [&](int t) { return __builtin_amdgcn_readlane(page_reg, page_n * NT + t); };
    u4 kf[2][NT][NK];
    const auto load_keys = [&](int step, int page[NT], u4 f[NT][NK]) {
#pragma unroll
        for (int t = 0; t < NT; t++) {
            page[t] = tile_page(t);
            const C* k = keys + paged_offset(a.p, max(page[t], 0), kvh, (lo + STEP * step + 16 * t) & slots) + (size_t)c * HD + (F32 ? 4 * g : 8 * g);
#pragma unroll
            for (int i = 0; i < NK; i++) f[t][i] = *reinterpret_cast<const u4*>(k + i * (F32 ? 16 : 32));
        }
    };

    int page[NT], next_page[NT] = {};
    const auto step_on = [&](int step, u4 (&kc)[NT][NK], u4 (&kn)[NT][NK]) {
        // values of this step, keys of the next
        Words<VW> vr[NT][4];
#pragma unroll
        for (int t = 0; t < NT; t++) {
            const C* v = values + paged_offset(a.p, max(page[t], 0), kvh, ((lo + STEP * step + 16 * t) & slots) + 4 * g) + (size_t)c * NJ;
#pragma unroll
            for (int i = 0; i < 4; i++) vr[t][i] = load_words<VW>(v + (size_t)i * HD);
        }
        if (step + 4 < steps) {
            if (++page_n == 64 / NT) {
                page_n = 0;
                page_reg = pages_from(step + 4);
            }
            load_keys(step + 4, next_page, kn);
        }
        // scores
        float s[NT][4];
#pragma unroll
        for (int t = 0; t < NT; t++) {
            vf4 d = {0.0f, 0.0f, 0.0f, 0.0f};
            if constexpr (F32) {
#pragma unroll
                for (int k = 0; k < NK; k++)
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        d = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(kc[t][k][e]), __uint_as_float(qf[0][k][e]), d, 0, 0, 0);
            } else {
#pragma unroll
                for (int p = NP - 1; p >= 0; p--)
#pragma unroll
                    for (int k = 0; k < NK; k++) d = T::mul(kc[t][k], qf[p][k], d);
            }
#pragma unroll
            for (int i = 0; i < 4; i++) s[t][i] = d[i] * unscale;
        }
        // positions that some row does not attend to
        const int p0 = lo + STEP * step;
        bool edge = p0 + STEP > min(least, hi);
#pragma unroll
        for (int t = 0; t < NT; t++) edge = edge || page[t] < 0;
        bool odd = false;      // a value that is no number at a position that some rows attend to
        if (edge) {
#pragma unroll
            for (int t = 0; t < NT; t++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int pos = p0 + 16 * t + 4 * g + i;
                    const bool held = page[t] >= 0 && pos < hi;
                    if (!held || pos >= lim) s[t][i] = -INFINITY;
#pragma unroll
                    for (int w = 0; w < VW; w++) {
                        if (!held) vr[t][i].w[w] = 0u;
                        if constexpr (F32) odd = odd || (vr[t][i].w[w] & 0x7f800000u) == 0x7f800000u;
                        else odd = odd || !T::finite(vr[t][i].w[w]);
                    }
                }
            odd = __ballot(odd) != 0 && p0 + STEP > least;
        }
        float mx = s[0][0];
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
            for (int i = 0; i < 4; i++) mx = fmaxf(mx, s[t][i]);
        if (__ballot(mx > m + kSlack)) {              // (m = -inf: any score raises it)
            const float m_new = fmaxf(m, group_max16(mx));
            const float alpha = m_new == m ? 1.0f : __builtin_amdgcn_exp2f(m - m_new);
            l *= alpha;
#pragma unroll
            for (int j = 0; j < NJ; j++) acc[j] *= alpha;
            m = m_new;
        }
        const float back = T::kBias - (m == -INFINITY ? 0.0f : m);
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                s[t][i] = __builtin_amdgcn_exp2f(s[t][i] + back);
                l += s[t][i];
            }
        if (odd) {
            // one position after the other, each only for the rows that attend to it
            for (int pos = 0; pos < STEP; pos++) {
                const int t = pos >> 4, from = ((pos >> 2) & 3) * 16 + c, i = pos & 3;
                float w = 0.0f;
#pragma unroll
                for (int tt = 0; tt < NT; tt++)
#pragma unroll
                    for (int ii = 0; ii < 4; ii++) {
                        const float got = __shfl(s[tt][ii], from, 64);
                        if (tt == t && ii == i) w = got;
                    }
                int pg = page[0];
#pragma unroll
                for (int tt = 1; tt < NT; tt++)
                    if (t == tt) pg = page[tt];
                if (pg < 0 || p0 + pos >= lim || p0 + pos >= hi) continue;
                const C* v = values + paged_offset(a.p, pg, kvh, (p0 + pos) & slots) + (size_t)4 * g * NJ;
#pragma unroll
                for (int ii = 0; ii < 4; ii++)
#pragma unroll
                    for (int j = 0; j < NJ; j++) acc[j][ii] = fmaf(w, (float)v[ii * NJ + j], acc[j][ii]);
            }
        } else if constexpr (F32) {
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int j = 0; j < NJ; j++)
                    acc[j] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(vr[0][i].w[j]), s[0][i], acc[j], 0, 0, 0);
        } else {
            u4 pf[NP];
#pragma unroll
            for (int d = 0; d < 4; d++) {
                uint32_t part[NP];
                T::cut(s[d >> 1][2 * (d & 1)], s[d >> 1][2 * (d & 1) + 1], part);
#pragma unroll
                for (int p = 0; p < NP; p++) pf[p][d] = part[p];
            }
#pragma unroll
            for (int j = 0; j < NJ; j++) {
                u4 vf;
#pragma unroll
                for (int d = 0; d < 4; d++)
                    vf[d] = __builtin_amdgcn_perm(vr[d >> 1][2 * (d & 1) + 1].w[j >> 1], vr[d >> 1][2 * (d & 1)].w[j >> 1],
                                                  j & 1 ? 0x07060302 : 0x05040100);
#pragma unroll
                for (int p = NP - 1; p >= 0; p--) acc[j] = T::mul(vf, pf[p], acc[j]);
            }
        }
#pragma unroll
        for (int t = 0; t < NT; t++) page[t] = next_page[t];
    };
    if (wave < steps) {
        load_keys(wave, page, kf[0]);
        for (int step = wave; step < steps; step += 8) {
            step_on(step, kf[0], kf[1]);
            if (step + 4 < steps) step_on(step + 4, kf[1], kf[0]);
        }
    }

    // the four wavefronts' results together
    l = group_sum16(l);
    if (g == 0) { sm[wave][c] = m; sl[wave][c] = l; }
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
        for (int j = 0; j < NJ; j++) so[wave][c][(4 * g + i) * NJ + j] = acc[j][i];
    __syncthreads();
    const int r = tid >> 4, e0 = (tid & 15) * NJ;      // row of the tile, NJ neighbouring dimensions
    float M = -INFINITY;
#pragma unroll
    for (int w = 0; w < 4; w++) M = fmaxf(M, sm[w][r]);
    float L = 0.0f, o[NJ] = {};
#pragma unroll
    for (int w = 0; w < 4; w++) {
        // (a wavefront without positions: weight 0; its sums are 0 or, with NaN scores only, NaN)
        const float f = sm[w][r] == M ? 1.0f : __builtin_amdgcn_exp2f(sm[w][r] - M);
        L = fmaf(sl[w][r], f, L);
#pragma unroll
        for (int k = 0; k < NJ; k++) o[k] = fmaf(so[w][r][e0 + k], f, o[k]);
    }
    const int sr = tile * kRowTile + r;
    if (sr >= set.rows * a.group) return;
    const int orow = set.first + sr / a.group, ohead = kvh * a.group + sr % a.group;
    if (whole) {
        const float inv = L != 0.0f ? 1.0f / L : 0.0f;
        float* dst = a.out + (size_t)orow * a.out_ld + (size_t)ohead * HD + e0;
#pragma unroll
        for (int k = 0; k < NJ; k++) dst[k] = o[k] * inv;
    } else {
        const size_t at = ((size_t)orow * a.p.n_heads + ohead) * a.parts + a.part0 + split;
        float* dst = a.po + at * HD + e0;
#pragma unroll
        for (int k = 0; k < NJ; k++) dst[k] = o[k];
        // (NaN scores alone leave the maximum at -inf: 0 marks the part as there)
        if ((tid & 15) == 0) a.pml[at] = make_float2(M == -INFINITY && L != 0.0f ? 0.0f : M, L);
    }
}

// Joins the partial results of one row and head: weights 2^(m - max), a
// quarter of the parts per wavefront, HD / 64 (or one) dimensions per lane.
template <int HD>
__global__ __launch_bounds__(256) void k_paged_attn_join(PagedAttn a) {
    constexpr int E = HD < 64 ? 1 : HD / 64;
    __shared__ float so[4][HD], sl[4], sm[4];
    const int row = blockIdx.x / a.p.n_heads, head = blockIdx.x % a.p.n_heads;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    if (a.p.row_start) {
        const int s = paged_seq_of_row(a.p, row);
        if (s < 0) return;
        int first, end;
        paged_rows(a.p, s, &first, &end);
        if (row < first || row >= end) return;
    }
    const float2* ml = a.pml + (size_t)blockIdx.x * a.parts;
    const float* po = a.po + (size_t)blockIdx.x * a.parts * HD;
    float M = -INFINITY;
    for (int i = tid; i < a.parts; i += 256) M = fmaxf(M, ml[i].x);
    for (int o = 32; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor(M, o, 64));
    if (lane == 0) sm[wave] = M;
    __syncthreads();
    M = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3]));
    float L = 0.0f, o[E] = {};
    for (int i = wave; i < a.parts; i += 4) {
        const float2 v = ml[i];
        if (v.x == -INFINITY) continue;
        const float f = __builtin_amdgcn_exp2f(v.x - M);
        L = fmaf(v.y, f, L);
#pragma unroll
        for (int e = 0; e < E; e++)
            if (HD >= 64 || lane < HD) o[e] = fmaf(po[(size_t)i * HD + E * lane + e], f, o[e]);
    }
    if (lane == 0) sl[wave] = L;
#pragma unroll
    for (int e = 0; e < E; e++)
        if (HD >= 64 || lane < HD) so[wave][E * lane + e] = o[e];
    __syncthreads();
    if (tid < HD) {
        L = (sl[0] + sl[1]) + (sl[2] + sl[3]);
        const float v = (so[0][tid] + so[1][tid]) + (so[2][tid] + so[3][tid]);
        a.out[(size_t)row * a.out_ld + (size_t)head * HD + tid] = L != 0.0f ? v / L : 0.0f;
    }
}

// ------------------------------------------------------------------- host

namespace {

// How a call is split, from what the host knows of it.
struct AttnPlan {
    int slots = 0, splits = 1, chunk = 0;            // own pages
    int prefix_tiles = 0, prefix_splits = 0, prefix_chunk = 0;
    int parts = 1;
    size_t bytes = 0;
};

AttnPlan plan_attention(const PagedArgs& p, uint32_t max_len) {
    AttnPlan r;
    const int group = p.n_heads / p.n_kv;
    const int64_t cap = paged_capacity(p);
    const int64_t longest = max_len && max_len < cap ? max_len : cap;
    const int own = (int)std::max<int64_t>(longest - p.prefix_len, 0);
    r.slots = p.row_start ? (int)(((int64_t)p.n_rows * group) / kRowTile) + p.n_seqs : p.n_seqs * ((group + kRowTile - 1) / kRowTile);
    const auto split = [&](int64_t tiles, int positions, int* splits, int* chunk) {
        const int64_t want = std::max<int64_t>(2048 / std::max<int64_t>(tiles, 1), 1);
        *splits = (int)std::clamp<int64_t>(want, 1, std::max(1, (positions + 255) / 256));
        *chunk = ((positions + *splits - 1) / *splits + 127) & ~127;
    };
    split((int64_t)r.slots * p.n_kv, own, &r.splits, &r.chunk);
    r.parts = r.splits;
    if (p.prefix_len) {
        r.prefix_tiles = (int)(((int64_t)p.n_rows * group + kRowTile - 1) / kRowTile);
        split((int64_t)r.prefix_tiles * p.n_kv, p.prefix_len, &r.prefix_splits, &r.prefix_chunk);
        r.parts += r.prefix_splits;
    }
    if (r.parts > 1) r.bytes = (size_t)p.n_rows * p.n_heads * r.parts * (p.hd + 2) * sizeof(float);
    return r;
}

template <typename C>
hipError_t launch_rows(const PagedAttn& a, int tiles, int prefix, hipStream_t s) {
    auto k = a.p.hd == 32 ? k_paged_attn_rows<C, 32> : a.p.hd == 64 ? k_paged_attn_rows<C, 64> : k_paged_attn_rows<C, 128>;
    hipLaunchKernelGGL(k, dim3((unsigned)tiles * a.p.n_kv, a.splits), dim3(256), 0, s, a, prefix);
    return hipGetLastError();
}
hipError_t launch_rows_of(int dtype, const PagedAttn& a, int tiles, int prefix, hipStream_t s) {
    return dtype == YL_T_F32 ? launch_rows<float>(a, tiles, prefix, s) : dtype == YL_T_F16 ? launch_rows<_Float16>(a, tiles, prefix, s)
                                                                                          : launch_rows<__bf16>(a, tiles, prefix, s);
}

yl_status refuse(const char* what, yl_status st = YL_ERR_ARG) {
    set_error(what);
    return st;
}

}  // namespace
}  // namespace yl

using namespace yl;

extern "C" {

size_t yl_paged_attention_workspace(const yl_paged_cache* cache, const yl_paged_batch* batch, uint32_t n_heads) {
    PagedArgs p{};
    if (paged_args(cache, batch, n_heads, &p) != YL_OK || !p.n_rows || !p.n_seqs) return 0;
    return plan_attention(p, batch->max_len).bytes;
}

yl_status yl_paged_attention(float* out, size_t out_ld, const float* q, size_t q_ld, const yl_paged_cache* cache,
                             const yl_paged_batch* batch, uint32_t n_heads, float attn_scale, void* workspace,
                             size_t workspace_bytes, void* stream) {
    PagedAttn a{};
    const yl_status st = paged_args(cache, batch, n_heads, &a.p);
    if (st != YL_OK) return st;
    if (!a.p.n_rows || !a.p.n_seqs) return YL_OK;
    if (!out || !q) return refuse("paged_attention: no q or no out");
    const size_t att = (size_t)n_heads * cache->head_size;
    if (q_ld < att || out_ld < att) return refuse("paged_attention: rows further apart than they are long");
    if (q == out && q_ld != out_ld) return refuse("paged_attention: in place, q_ld and out_ld are the same");
    const AttnPlan plan = plan_attention(a.p, batch->max_len);
    if (plan.bytes && (!workspace || (uintptr_t)workspace % 16)) return refuse("paged_attention: the workspace has to be there, 16-byte aligned");
    if (workspace_bytes < plan.bytes) return refuse("paged_attention: the workspace is smaller than yl_paged_attention_workspace says", YL_ERR_RANGE);
    a.out = out; a.q = q; a.out_ld = out_ld; a.q_ld = q_ld;
    a.scale_log2 = attn_scale * 1.4426950408889634f;
    a.group = a.p.n_heads / a.p.n_kv;
    a.parts = plan.parts;
    a.po = static_cast<float*>(workspace);
    a.pml = reinterpret_cast<float2*>(a.po + (size_t)a.p.n_rows * a.p.n_heads * plan.parts * a.p.hd);
    hipStream_t s = (hipStream_t)stream;
    a.splits = plan.splits; a.chunk = plan.chunk; a.part0 = 0;
    hipError_t e = launch_rows_of(cache->dtype, a, plan.slots, 0, s);
    if (e == hipSuccess && plan.prefix_tiles) {
        a.splits = plan.prefix_splits; a.chunk = plan.prefix_chunk; a.part0 = plan.splits;
        e = launch_rows_of(cache->dtype, a, plan.prefix_tiles, 1, s);
    }
    if (e == hipSuccess && plan.parts > 1) {
        auto k = a.p.hd == 32 ? k_paged_attn_join<32> : a.p.hd == 64 ? k_paged_attn_join<64> : k_paged_attn_join<128>;
        hipLaunchKernelGGL(k, dim3((unsigned)a.p.n_rows * a.p.n_heads), dim3(256), 0, s, a);
        e = hipGetLastError();
    }
    if (e == hipSuccess) return YL_OK;
    set_error(std::string("paged_attention launch: ") + hipGetErrorString(e));
    return YL_ERR_HIP;
}

}  // extern "C"
