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
// by dimension: from registers (row kernel) a lane loads HD / 16 neighbouring
// dimensions of its 8 positions and picks each dimension's halves with v_perm, no
// lane exchange; from LDS (tile kernel) transposing reads bring it as it is wanted.
//
// Kernels of a call, in the stream's order: the row kernel (sequences of few
// rows, every f32 call), the tile kernel (sequences of many rows), one of the
// two over a shared prefix, and a join of partial results where there are any.
//
// Precision: the products run on f16 / bf16 matrix instructions with f32 sums
// while q and the weights are f32, so these are cut into parts that add up to
// them: two f16 (22 bits; q scaled per row by a power of two, the weights against a
// reference, so that the second part keeps its bits) or three bf16 (24 bits; two
// would leave errors of 2^-18 of a weight).  f32 caches take the f32 matrix
// instructions.
//
// Softmax: running reference and sum per row in base 2 (one pass over the keys);
// the weight of a score is 2^(score - reference).  The reference is the largest
// score less the type's bias when it is set, and is only raised when a weight
// would pass 2^kMost, so that most steps need no exchange between lanes and no
// rescaling.  Over f16 caches it also falls, by up to some 40 powers of two, where
// all of a step's weights would be below 2^kLeast: f16 parts end at 2^-24, and
// beside one position that has nearly all of the weight the others would lose
// their bits.  Scores come out of the products times a power of two (the scale's
// mantissa is multiplied into q), so that one fma subtracts the reference from
// the score itself: a product rounded on its way would be off by many powers of
// two where scores are large.
#include <hip/hip_runtime.h>

#include <math.h>

#include <algorithm>
#include <cmath>

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

// What depends on the cache's type.
template <typename C> struct Type;
template <> struct Type<_Float16> {
    static constexpr uint32_t kOnes = 0x3c003c00u;
    static constexpr int kParts = 2, kTiles = 2;   // parts of an f32 value; 16-position tiles of one step
    // The largest weight of a step is between 2^-2 and 2^15 (2^11 when the
    // reference is raised, 2^7 when it falls): a weight has 22 bits, and what is
    // below 2^-2 is right to 2^-25, at most 2^-23 of the step's largest.  A prompt
    // of 5280 tokens, hd 64, without falls | with kLeast 1 | -2 | -4, in us: scores of
    // deviation 1 258.7 | 257.9 | 257.8 | 258.0, 2 258.6 | 262.1 | 260.3 | 259.9, 3 257.0 |
    // 275.8 | 268.5 | 263.3.
    static constexpr bool kFalls = true;
    static constexpr float kBias = 11.0f, kMost = 15.0f, kLeast = -2.0f, kFall = 7.0f;
    static constexpr int kRoom = 52;               // sums of weights are left below 2^52 by a fall
    static __device__ __forceinline__ vf4 mul(u4 a, u4 b, vf4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c, 0, 0, 0);
    }
    // two values -> their parts, packed
    static __device__ __forceinline__ void cut(float a, float b, uint32_t part[2]) {
        const h2 hi = __builtin_convertvector(vf2{a, b}, h2);
        part[0] = __builtin_bit_cast(uint32_t, hi);
        // a - hi, b - hi rounded to f16: one mixed-precision fma each
        asm("v_fma_mixlo_f16 %0, %1, -1.0, %2 op_sel_hi:[1,0,0]\n\tv_fma_mixhi_f16 %0, %1, -1.0, %3 op_sel:[1,0,0] op_sel_hi:[1,0,0]"
            : "=&v"(part[1]) : "v"(part[0]), "v"(a), "v"(b));
    }
    // the power of two that brings a row of q to [2^13, 2^14): its elements keep
    // 22 bits down to 2^-15 of the largest, and are right to 2^-38 of it below
    static __device__ __forceinline__ int exponent(float amax) {
        return amax > 0.0f && amax < INFINITY ? min(14 - __builtin_amdgcn_frexp_expf(amax), 110) : 0;
    }
    // all bits of the halves that are no numbers
    static __device__ __forceinline__ uint32_t not_finite(uint32_t two) {
        return ((two & 0x7c00u) == 0x7c00u ? 0xffffu : 0u) | ((two & 0x7c000000u) == 0x7c000000u ? 0xffff0000u : 0u);
    }
};
template <> struct Type<__bf16> {
    static constexpr uint32_t kOnes = 0x3f803f80u;
    static constexpr int kParts = 3, kTiles = 2;
    static constexpr bool kFalls = false;
    static constexpr float kBias = 0.0f, kMost = 8.0f;
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
    static __device__ __forceinline__ uint32_t not_finite(uint32_t two) {
        return ((two & 0x7f80u) == 0x7f80u ? 0xffffu : 0u) | ((two & 0x7f800000u) == 0x7f800000u ? 0xffff0000u : 0u);
    }
};
template <> struct Type<float> {
    static constexpr int kParts = 1, kTiles = 1;
    static constexpr bool kFalls = false;
    static constexpr float kBias = 0.0f, kMost = 8.0f;
    static __device__ __forceinline__ uint32_t not_finite(uint32_t x) { return (x & 0x7f800000u) == 0x7f800000u ? ~0u : 0u; }
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
// the largest of 16 neighbouring lanes (every lane active)
__device__ __forceinline__ int max16(int v) {
    v = max(v, __builtin_amdgcn_update_dpp(v, v, 0xB1, 0xF, 0xF, false));    // quad_perm [1,0,3,2]
    v = max(v, __builtin_amdgcn_update_dpp(v, v, 0x4E, 0xF, 0xF, false));    // quad_perm [2,3,0,1]
    v = max(v, __builtin_amdgcn_update_dpp(v, v, 0x141, 0xF, 0xF, false));   // row_half_mirror
    return max(v, __builtin_amdgcn_update_dpp(v, v, 0x140, 0xF, 0xF, false)); // row_mirror
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
    float scale; int scale_exp;      // attn_scale * log2(e) = scale * 2^scale_exp, 0.5 <= |scale| < 1
    int group;                       // query heads per kv head
    int parts, part0;                // partial results per row and head; the first of this launch's
    int chunk;                       // positions of a split at least
    int splits;
    int direct;                      // this launch sees all that its rows attend to: it writes `out`
    // the row kernel's own work: units wanted, beyond one per tile, and units
    // there is room for; where each sequence's units begin and how many its
    // tiles have, for the joining kernel.  wanted 0: positions not split, a unit
    // for each slot of `per` per sequence of one row, or as of tile_of_slot
    int per, wanted, max_units;
    float finer;                     // units wanted per tile where there are many tiles
    int4* units;
    int joined;                      // the joining kernel follows
    int both;                        // sequences are divided between the row kernel and the tile kernel
    // partial results, unnormalised, and their reference (base 2) and sum, reference
    // -inf: nothing there.  Of the row kernel's own work [unit][n_kv][16 rows],
    // of the others [row][n_heads][parts]
    float* po;
    float2* pml;
};

// A tile of the stacked rows that attend to the same pages.
struct RowSet {
    const int32_t* pages; int entries;   // entry of position i: pages[i >> page_shift], i < entries << page_shift
    int first, rows;                     // rows of the batch; stacked row i is row first + i / group
    int seq;                             // sequence, or -1: the whole batch over the prefix
};

__device__ __forceinline__ RowSet set_of_seq(const PagedArgs& p, int seq) {
    RowSet set;
    set.seq = seq;
    set.entries = p.max_pages;
    set.pages = p.table + (size_t)seq * p.max_pages;
    int end;
    paged_rows(p, seq, &set.first, &end);
    set.rows = end - set.first;
    return set;
}

// The tile of slot `slot`: sequence s takes slots from floor(row_start[s] *
// group / rows of a tile) + s on, of which it uses one per tile: a sequence's
// slots always suffice, and are found by a search over row_start alone (64
// starts per step, one per lane).  False: a slot that nothing uses.
__device__ __forceinline__ int first_slot(const PagedAttn& a, int s, int rows_log2) {
    const uint32_t st = a.p.row_start[s];
    return (int)(((int64_t)(st < (uint32_t)a.p.n_rows ? (int)st : a.p.n_rows) * a.group) >> rows_log2) + s;
}
__device__ __forceinline__ bool tile_of_slot(const PagedAttn& a, int slot, int rows_log2, RowSet* set, int* tile) {
    const PagedArgs& p = a.p;
    const int lane = threadIdx.x & 63;
    const auto base = [&](int s) { return first_slot(a, s, rows_log2); };
    int lo = 0, n = p.n_seqs;
    while (n > 1) {
        const int step = (n + 63) >> 6;
        const bool ok = lane * step < n && base(lo + lane * step) <= slot;
        const int c = max(1, (int)__builtin_popcountll(__ballot(ok))) - 1;
        lo += c * step;
        n = min(step, n - c * step);
    }
    lo = __builtin_amdgcn_readfirstlane(lo);
    *set = set_of_seq(p, lo);
    *tile = slot - base(lo);
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

constexpr int kRowTile = 16, kRowTileLog2 = 4;

// Stacked rows of a sequence (tokens times heads per kv head) up to which the
// row kernel takes it where there is work for the tile kernel.  64 turns of so many
// stacked rows beside a prompt of 1500 tokens, 32 heads on 8, in us, row kernel |
// tile kernel:
//   stacked rows               24             32             40             64
//   f16 hd 64,  300 long   73.6 | 61.5    75.0 | 62.5    83.9 | 69.8    81.7 | 70.7
//              2000 long    122 | 107      126 | 107      145 | 113      156 | 114
//   bf16 hd 128, 300 long   116 | 116      117 | 117      134 | 131      146 | 125
//              2000 long                   207 | 226      242 | 266      274 | 243
constexpr int kRowKernelRows = 32;
__device__ __forceinline__ bool row_kernel_takes(int rows, int group) { return (int64_t)rows * group <= kRowKernelRows; }

// A unit of the row kernel's own work: a tile of a sequence's rows over one of
// `splits` stretches of its positions.  `first`: the sequence's first unit.
struct Unit {
    int seq, tile, split, splits, chunk, first;
};

__device__ __forceinline__ int scan_add(int x) {       // inclusive, over the 64 lanes
    x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xF, 0xF, true);
    x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xF, 0xF, true);
    x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xF, 0xF, true);
    x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xF, 0xF, true);
    x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xA, 0xF, true);
    x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xC, 0xF, true);
    return x;
}

__device__ __forceinline__ float wave_sum(float x) {   // every lane active
    x += dpp_mov<0xB1>(x);
    x += dpp_mov<0x4E>(x);
    x += dpp_mov<0x141>(x);
    x += dpp_mov<0x140>(x);
    return (lane_value(x, 0) + lane_value(x, 16)) + (lane_value(x, 32) + lane_value(x, 48));
}

// Sequences up to which their work is divided by their lengths: beyond it there
// are workgroups enough, and the kernel finds its tile by a search.  32 heads on
// 8, hd 64, f16, one row each, divided | not, in us: 512 of 100 .. 8000 positions
// 373 | 407, of 100 .. 3000 208 | 194; 1024 of them 721 | 707, 405 | 338.
constexpr int kDivided = 512;

// Unit `u` of the batch.  All tiles' positions together, divided by the units
// wanted, are a unit's share: a long sequence becomes many units, a short one
// one, whatever the lengths are when the work runs.  Every wavefront works
// this out from the lengths, alike (all of them in flight at once: as two loops
// of 64 a step 512 sequences of 100 .. 3000 took 251).
__device__ __forceinline__ bool unit_of(const PagedAttn& a, int u, Unit* r) {
    constexpr int K = kDivided / 64;
    const PagedArgs& p = a.p;
    const int lane = threadIdx.x & 63, steps = (p.n_seqs + 63) >> 6;
    // sequences' tiles (none where the tile kernel takes them) and their longest rows' positions
    int tiles[K], len[K];
    float sum = 0.0f, all = 0.0f;
#pragma unroll
    for (int k = 0; k < K; k++) {
        const int s = 64 * k + lane;
        tiles[k] = len[k] = 0;
        if (k >= steps || s >= p.n_seqs) continue;
        int first, end;
        paged_rows(p, s, &first, &end);
        const int n = end - first, held = max(paged_limit(p, (int64_t)p.kv_len[s] - 1) - p.prefix_len, 0);
        if (n == 0 || (a.both && !row_kernel_takes(n, a.group))) continue;
        tiles[k] = (n * a.group + kRowTile - 1) / kRowTile;
        len[k] = held;
        sum += (float)tiles[k] * (float)held;
        all += (float)tiles[k];
    }
    sum = wave_sum(sum);
    all = wave_sum(all);
    // (rounded up beyond the sum's own rounding, so that the units never are more than there is room for)
    const float share = sum * 1.001f / fmaxf((float)a.wanted, a.finer * all);
    const int chunk = share < 1e9f && a.chunk < 1 << 30 ? (max((int)share + 1, a.chunk) + 63) & ~63 : 1 << 30;
    int before = 0;
#pragma unroll
    for (int k = 0; k < K; k++) {
        if (k >= steps) break;
        const int splits = max(1, (int)(((unsigned)len[k] + (unsigned)chunk - 1u) / (unsigned)chunk));
        const int mine = tiles[k] * splits, upto = before + scan_add(mine);
        const auto here = __ballot(u < upto);
        if (here) {
            const int l = __builtin_ctzll(here);
            r->seq = 64 * k + l;
            r->splits = __builtin_amdgcn_readlane(splits, l);
            r->first = __builtin_amdgcn_readlane(upto - mine, l);
            const int i = u - r->first;
            if (i < 0) return false;                       // (starts that do not ascend)
            r->tile = i / r->splits;
            r->split = i - r->tile * r->splits;
            r->chunk = chunk;
            return true;
        }
        before = __builtin_amdgcn_readlane(upto, 63);
    }
    return false;
}

// 16 stacked rows in a wavefront: lane (c, g) holds of row c the query parts,
// the sums acc[j][i] of dimensions dim(i, j) and those of its positions.
// TR: V^T's operands come transposed from LDS (f16 and bf16), a lane's
// dimensions are 16 apart, and a matrix product with ones adds up the weights;
// otherwise from whole rows in registers, NJ neighbouring dimensions per lane.
template <typename C, int HD, bool TR>
struct Tile {
    using T = Type<C>;
    static constexpr bool F32 = sizeof(C) == 4;
    static constexpr int NT = T::kTiles, NP = T::kParts, STEP = 16 * NT;
    static constexpr int NJ = HD / 16;                       // dimensions per lane of V, tiles of O^T
    static constexpr int NK = F32 ? HD / 16 : HD / 32;       // 16-byte pieces of a key per lane
    static constexpr int KD = F32 ? 16 : 32, KE = F32 ? 4 : 8;   // dimensions per piece of all lane groups, of one
    static constexpr int VW = NJ * (int)sizeof(C) / 4;       // words of a V row per lane
    static_assert(!(TR && F32), "halfwords are transposed");
    typedef Words<VW> Value;
    static __device__ __forceinline__ int dim(int i, int j, int g) { return TR ? 16 * j + 4 * g + i : (4 * g + i) * NJ + j; }

    int row, head, lim;              // lim: positions below it are attended to
    bool live;
    float m, l, unscale;             // m: the weights' reference
    u4 qf[NP][NK];
    vf4 acc[NJ], ones;               // ones: sums of the weights (TR)

    // Places the tile at stacked rows from `stacked` on.
    __device__ __forceinline__ void place(const PagedAttn& a, const RowSet& set, int stacked, int kvh, int c) {
        const int r = stacked + c;
        live = r < set.rows * a.group;
        row = set.first + (live ? r / a.group : 0);
        head = kvh * a.group + (live ? r % a.group : 0);
        m = -INFINITY;
        l = 0.0f;
#pragma unroll
        for (int j = 0; j < NJ; j++) acc[j] = vf4{0.0f, 0.0f, 0.0f, 0.0f};
        ones = vf4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    // The sum of row c's weights, in every lane of the row (!TR: before they are
    // cut, which is within their parts' own rounding).
    __device__ __forceinline__ float sum() const { return TR ? ones[0] : group_sum16(l); }
    // What the rows attend to, and the longest and the shortest of them
    // (spare rows follow the longest, so that they need no masks).
    __device__ __forceinline__ void reach(const PagedAttn& a, const RowSet& set, int* most, int* least) {
        lim = live ? (int)min((int64_t)limit_of_row(a, set, row), (int64_t)set.entries << a.p.page_shift) : 0;
        *most = __builtin_amdgcn_readfirstlane(max16(lim));
        if (!live) lim = *most;
        *least = -__builtin_amdgcn_readfirstlane(max16(-lim));
    }
    // q of the lane's row, cut into parts, in the order of the keys' pieces
    __device__ __forceinline__ void load_q(const PagedAttn& a, int g) {
        const float* qr = a.q + (size_t)row * a.q_ld + (size_t)head * HD + KE * g;
        f4u v[NK][KE / 4];
        float amax = 0.0f;
#pragma unroll
        for (int k = 0; k < NK; k++)
#pragma unroll
            for (int e = 0; e < KE / 4; e++) {
                v[k][e] = *reinterpret_cast<const f4u*>(qr + k * KD + 4 * e);
                if (!live) v[k][e] = f4u{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int i = 0; i < 4; i++) amax = fmaxf(amax, fabsf(v[k][e][i]));
            }
        // scores times `unscale`, a power of two, are the exponents
#pragma unroll
        for (int k = 0; k < NK; k++)
#pragma unroll
            for (int e = 0; e < KE / 4; e++) v[k][e] *= a.scale;
        int ex = 0;
        if constexpr (F32) {
#pragma unroll
            for (int k = 0; k < NK; k++) qf[0][k] = __builtin_bit_cast(u4, v[k][0]);
        } else {
            ex = T::exponent(group_max16(amax * fabsf(a.scale)));
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
        unscale = __builtin_amdgcn_ldexpf(1.0f, min(max(a.scale_exp - ex, -126), 127));
    }
    // scores of the step's positions, before `unscale` (the tiles' chains of products side by side)
    __device__ __forceinline__ void scores(const u4 kc[NT][NK], float s[NT][4]) const {
        vf4 d[NT];
#pragma unroll
        for (int t = 0; t < NT; t++) d[t] = vf4{0.0f, 0.0f, 0.0f, 0.0f};
        if constexpr (F32) {
#pragma unroll
            for (int k = 0; k < NK; k++)
#pragma unroll
                for (int e = 0; e < 4; e++)
                    d[0] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(kc[0][k][e]), __uint_as_float(qf[0][k][e]), d[0], 0, 0, 0);
        } else {
#pragma unroll
            for (int p = NP - 1; p >= 0; p--)
#pragma unroll
                for (int k = 0; k < NK; k++)
#pragma unroll
                    for (int t = 0; t < NT; t++) d[t] = T::mul(kc[t][k], qf[p][k], d[t]);
        }
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
            for (int i = 0; i < 4; i++) s[t][i] = d[t][i];
    }
    // Takes positions that are not there, or past the row, out of the scores.
    __device__ __forceinline__ void mask(float s[NT][4], int p0, int hi, const int page[NT], int g) const {
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int pos = p0 + 16 * t + 4 * g + i;
                if (page[t] < 0 || pos >= min(lim, hi)) s[t][i] = -INFINITY;
            }
    }
    // scores -> weights of N tiles of positions, under a reference that is raised where it has to be
    template <int N>
    __device__ __forceinline__ void weigh(float (*s)[4]) {
        float mx = s[0][0];
#pragma unroll
        for (int t = 0; t < N; t++)
#pragma unroll
            for (int i = 0; i < 4; i++) mx = fmaxf(mx, s[t][i]);
        const float e = fmaf(mx, unscale, -m);               // (m = -inf: any score raises it)
        bool off = e > T::kMost;
        if constexpr (T::kFalls) off = !(e >= T::kLeast && e <= T::kMost);
        if (__ballot(off)) {
            const float top = group_max16(mx) * unscale;
            float to = fmaxf(m, top - T::kBias);
            // (where floats are further apart than the bias)
            if (T::kBias > 0.0f && top - to > T::kMost) to = top;
            if constexpr (T::kFalls) {
                const bool low = top - m < T::kLeast && top > -INFINITY && fabsf(m) < 0x1p20f;   // (beyond it scores are not this exact)
                if (__ballot(low)) {
                    const int room = max(T::kRoom - __builtin_amdgcn_frexp_expf(sum()), 0);
                    if (low) to = fmaxf(top - T::kFall, m - (float)room);
                }
            }
            const float alpha = to == m ? 1.0f : __builtin_amdgcn_exp2f(m - to);
            if constexpr (TR) ones *= alpha;
            else l *= alpha;
#pragma unroll
            for (int j = 0; j < NJ; j++) acc[j] *= alpha;
            m = to;
        }
        const float ref = m == -INFINITY ? 0.0f : m;
#pragma unroll
        for (int t = 0; t < N; t++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                s[t][i] = __builtin_amdgcn_exp2f(fmaf(s[t][i], unscale, -ref));
                if constexpr (!TR) l += s[t][i];
            }
    }
    // V^T's operands: of f16 and bf16, dimension j's halves of the 8 positions
    static __device__ __forceinline__ u4 operand(const Value vr[NT][4], int j) {
        u4 f;
#pragma unroll
        for (int d = 0; d < 4; d++)
            f[d] = __builtin_amdgcn_perm(vr[d >> 1][2 * (d & 1) + 1].w[j >> 1], vr[d >> 1][2 * (d & 1)].w[j >> 1],
                                         j & 1 ? 0x07060302 : 0x05040100);
        return f;
    }
    // adds the weighted values
    __device__ __forceinline__ void add(const float s[NT][4], const Value vr[NT][4]) {
        if constexpr (F32) {
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int j = 0; j < NJ; j++)
                    acc[j] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(vr[0][i].w[j]), s[0][i], acc[j], 0, 0, 0);
        } else {
            u4 vf[NJ];
#pragma unroll
            for (int j = 0; j < NJ; j++) vf[j] = operand(vr, j);
            add(s, vf);
        }
    }
    __device__ __forceinline__ void add(const float s[NT][4], const u4 vf[NJ]) {
        u4 pf[NP];
#pragma unroll
        for (int d = 0; d < 4; d++) {
            uint32_t part[NP];
            T::cut(s[d >> 1][2 * (d & 1)], s[d >> 1][2 * (d & 1) + 1], part);
#pragma unroll
            for (int p = 0; p < NP; p++) pf[p][d] = part[p];
        }
#pragma unroll
        for (int p = NP - 1; p >= 0; p--) {
            if constexpr (TR) ones = T::mul(u4{T::kOnes, T::kOnes, T::kOnes, T::kOnes}, pf[p], ones);
#pragma unroll
            for (int j = 0; j < NJ; j++) acc[j] = T::mul(vf[j], pf[p], acc[j]);
        }
    }
    // Adds the values that are no numbers (clear_values has taken them out)
    // where rows differ in what they attend to: as 0 times one of them is no
    // number either, only to the rows that attend to its position.
    __device__ __forceinline__ void add_odd(const PagedAttn& a, const float s[NT][4], int p0, int hi, const int page[NT], int kvh, int c, int g) {
        const int slots = (1 << a.p.page_shift) - 1;
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
            if (pg < 0 || p0 + pos >= min(lim, hi)) continue;
            const C* v = static_cast<const C*>(a.p.values) + paged_offset(a.p, pg, kvh, (p0 + pos) & slots);
#pragma unroll
            for (int ii = 0; ii < 4; ii++)
#pragma unroll
                for (int j = 0; j < NJ; j++) {
                    const float x = (float)v[dim(ii, j, g)];
                    if (!(fabsf(x) < INFINITY)) acc[j][ii] = fmaf(w, x, acc[j][ii]);
                }
        }
    }
};

// Clears values that are not there, and among positions that not every row
// attends to those that are no numbers; true if there was one of the latter.
template <typename C, int HD>
__device__ __forceinline__ bool clear_values(typename Tile<C, HD, false>::Value vr[Tile<C, HD, false>::NT][4], int p0, int hi,
                                             bool differ, const int page[], int g) {
    using R = Tile<C, HD, false>;
    uint32_t odd = 0;
#pragma unroll
    for (int t = 0; t < R::NT; t++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const bool held = page[t] >= 0 && p0 + 16 * t + 4 * g + i < hi;
#pragma unroll
            for (int w = 0; w < R::VW; w++) {
                uint32_t x = held ? vr[t][i].w[w] : 0u;
                if (differ) {
                    const uint32_t bad = R::T::not_finite(x);
                    odd |= bad;
                    x &= ~bad;
                }
                vr[t][i].w[w] = x;
            }
        }
    return __ballot(odd != 0) != 0;
}

// The same of transposed operands: word d of each holds positions 16 (d / 2) + 4g + 2 (d % 2) and the next.
template <typename C, int HD>
__device__ __forceinline__ bool clear_operands(u4 vf[HD / 16], int p0, int hi, bool differ, const int page[2], int g) {
    uint32_t odd = 0;
#pragma unroll
    for (int d = 0; d < 4; d++) {
        const int pos = p0 + 16 * (d >> 1) + 4 * g + 2 * (d & 1), n = page[d >> 1] >= 0 ? hi - pos : 0;
        const uint32_t held = n >= 2 ? ~0u : n == 1 ? 0xffffu : 0u;
#pragma unroll
        for (int j = 0; j < HD / 16; j++) {
            uint32_t x = vf[j][d] & held;
            if (differ) {
                const uint32_t bad = Type<C>::not_finite(x);
                odd |= bad;
                x &= ~bad;
            }
            vf[j][d] = x;
        }
    }
    return __ballot(odd != 0) != 0;
}

// The stretch [lo, hi) of positions that a split covers, of the `most` that a tile attends to.
__device__ __forceinline__ void split_range(const PagedAttn& a, int split, int most, int* lo, int* hi) {
    *lo = 0;
    *hi = most;
    if (a.splits > 1) {
        const int even = (most + a.splits - 1) / a.splits;
        const int chunk = max(a.chunk, (even + 63) & ~63);
        *lo = (int)min((int64_t)split * chunk, (int64_t)most);
        *hi = most - *lo < chunk ? most : *lo + chunk;
    }
}

// The prefix as every row's pages.
__device__ __forceinline__ RowSet prefix_set(const PagedAttn& a) {
    return RowSet{a.p.prefix_pages, (a.p.prefix_len + (1 << a.p.page_shift) - 1) >> a.p.page_shift, 0, a.p.n_rows, -1};
}

// Where a row's partial result of the tile kernel, or over the prefix, stands.
__device__ __forceinline__ size_t part_of(const PagedAttn& a, int row, int head, int split) {
    return ((size_t)row * a.p.n_heads + head) * a.parts + a.part0 + split;
}

// One tile of 16 stacked rows over one stretch of the positions, the positions
// dealt to four wavefronts in steps of 16 NT.  K and V go from memory to
// registers in the operands' order; the next step's keys are loaded while
// this one is computed.  Bound by memory where there are workgroups enough: two
// rows at 128,000 positions, 32 heads on 8, f16, hd 64: 91 us, 5.8 TB/s; 64 rows
// at 100 .. 8000, bf16, hd 128: 122 us, 5.3 TB/s (units of unlike lengths).  A
// single row at 600 positions 8 us: launch, three round trips, then what one CU
// loads (57 GB/s); eight wavefronts for four, or values a step ahead, the same.
template <typename C, int HD>
__global__ __launch_bounds__(256, 2) void k_paged_attn_rows(PagedAttn a, int prefix) {
    using R = Tile<C, HD, false>;
    constexpr int NT = R::NT, NK = R::NK, NJ = R::NJ, STEP = R::STEP, LD = HD + 4, W = 4;
    __shared__ __align__(16) float so[4][kRowTile][LD];
    __shared__ float sm[4][kRowTile], sl[4][kRowTile];

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int c = lane & 15, g = lane >> 4;
    const int kvh = blockIdx.x % a.p.n_kv, slot = blockIdx.x / a.p.n_kv;
    RowSet set;
    Unit u{0, slot, (int)blockIdx.y, 1, 0, 0};     // (own pages: the grid is flat)
    if (prefix) {
        set = prefix_set(a);
    } else {
        if (a.wanted) {
            if (!unit_of(a, slot, &u)) return;
            if (a.joined && slot == u.first && kvh == 0 && tid == 0) a.units[u.seq] = make_int4(u.first, u.splits, 0, 0);
        } else if (a.p.row_start) {
            if (!tile_of_slot(a, slot, kRowTileLog2, &set, &u.tile)) return;
            u.seq = set.seq;
            u.first = slot - u.tile;
        } else {
            u.seq = slot / a.per;
            u.first = u.seq * a.per;
            u.tile = slot - u.first;
        }
        set = set_of_seq(a.p, u.seq);
        if ((int64_t)(uint32_t)u.tile * kRowTile >= (int64_t)set.rows * a.group || (a.both && !row_kernel_takes(set.rows, a.group))) return;
    }
    const bool direct = a.direct && u.splits == 1;
    R r;
    r.place(a, set, u.tile * kRowTile, kvh, c);
    // Pages of this wavefront's next 64 tiles, one per lane (-1: none).  The
    // first are loaded from where the stretch begins if it begins where the
    // host's knowledge says, so that they, q and the lengths come in one round trip.
    const int64_t held = (int64_t)set.entries << a.p.page_shift;
    const auto pages_from = [&](int begin, int step) {
        const int64_t at = (int64_t)begin + STEP * (step + W * (lane / NT)) + 16 * (lane % NT);
        return at < held ? paged_page(set.pages[at >> a.p.page_shift], a.p.n_pages) : -1;
    };
    const int begin = (int)min((int64_t)u.split * (prefix ? a.chunk : u.chunk), held);
    int page_reg = pages_from(begin, wave), page_n = 0;
    r.load_q(a, g);
    int most, least, lo, hi;
    r.reach(a, set, &most, &least);
    if (prefix) {
        split_range(a, u.split, most, &lo, &hi);
    } else {
        lo = min(begin, most);
        hi = u.splits > 1 && most - lo > u.chunk ? lo + u.chunk : most;
    }
    // where the partial result of the tile's row `k` stands
    const auto part_at = [&](int k, int row, int head) {
        return prefix ? part_of(a, row, head, u.split) : ((size_t)slot * a.p.n_kv + kvh) * kRowTile + k;
    };
    if (lo >= hi && !direct) {
        if (r.live && wave == 0 && g == 0) a.pml[part_at(c, r.row, r.head)] = make_float2(-INFINITY, 0.0f);
        return;
    }
    if (lo != begin) page_reg = pages_from(lo, wave);

    const C* keys = static_cast<const C*>(a.p.keys);
    const C* values = static_cast<const C*>(a.p.values);
    const int slots = (1 << a.p.page_shift) - 1;
    const int steps = (hi - lo + STEP - 1) / STEP;
    u4 kf[2][NT][NK];
    const auto load_keys = [&](int step, int page[NT], u4 f[NT][NK]) {
#pragma unroll
        for (int t = 0; t < NT; t++) {
            const int got = __builtin_amdgcn_readlane(page_reg, page_n * NT + t);
            page[t] = lo + STEP * step + 16 * t < hi ? got : -1;
            const C* k = keys + paged_offset(a.p, max(page[t], 0), kvh, (lo + STEP * step + 16 * t) & slots) + (size_t)c * HD + R::KE * g;
#pragma unroll
            for (int i = 0; i < NK; i++) f[t][i] = *reinterpret_cast<const u4*>(k + i * R::KD);
        }
    };
    int page[NT], next_page[NT] = {};
    const auto step_on = [&](int step, u4 (&kc)[NT][NK], u4 (&kn)[NT][NK]) {
        // values of this step, keys of the next (the next step's values too
        // measured the same or, with a wavefront per SIMD fewer, slower)
        typename R::Value vr[NT][4];
#pragma unroll
        for (int t = 0; t < NT; t++) {
            const C* v = values + paged_offset(a.p, max(page[t], 0), kvh, ((lo + STEP * step + 16 * t) & slots) + 4 * g) + (size_t)c * NJ;
#pragma unroll
            for (int i = 0; i < 4; i++) vr[t][i] = load_words<R::VW>(v + (size_t)i * HD);
        }
        if (step + W < steps) {
            if (++page_n == 64 / NT) {
                page_n = 0;
                page_reg = pages_from(lo, step + W);
            }
            load_keys(step + W, next_page, kn);
        }
        float s[NT][4];
        r.scores(kc, s);
        const int p0 = lo + STEP * step;
        bool edge = p0 + STEP > min(least, hi), odd = false;
#pragma unroll
        for (int t = 0; t < NT; t++) edge = edge || page[t] < 0;
        if (edge) {
            r.mask(s, p0, hi, page, g);
            odd = clear_values<C, HD>(vr, p0, hi, p0 + STEP > least, page, g);
        }
        r.template weigh<NT>(s);
        r.add(s, vr);
        if (odd) r.add_odd(a, s, p0, hi, page, kvh, c, g);
#pragma unroll
        for (int t = 0; t < NT; t++) page[t] = next_page[t];
    };
    if (wave < steps) {
        load_keys(wave, page, kf[0]);
        for (int step = wave; step < steps; step += 2 * W) {
            step_on(step, kf[0], kf[1]);
            if (step + W < steps) step_on(step + W, kf[1], kf[0]);
        }
    }

    // the wavefronts' results together
    const float l = r.sum();
    if (g == 0) { sm[wave][c] = r.m; sl[wave][c] = l; }
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
        for (int j = 0; j < NJ; j++) so[wave][c][R::dim(i, j, g)] = r.acc[j][i];
    __syncthreads();
    const int tr = tid >> 4, e0 = (tid & 15) * NJ;      // row of the tile, NJ neighbouring dimensions
    float M = -INFINITY;
#pragma unroll
    for (int w = 0; w < 4; w++) M = fmaxf(M, sm[w][tr]);
    float L = 0.0f, o[NJ] = {};
#pragma unroll
    for (int w = 0; w < 4; w++) {
        // (a wavefront without positions: weight 0; its sums are 0 or, with NaN scores only, NaN)
        const float f = sm[w][tr] == M ? 1.0f : __builtin_amdgcn_exp2f(sm[w][tr] - M);
        L = fmaf(sl[w][tr], f, L);
#pragma unroll
        for (int k = 0; k < NJ; k++) o[k] = fmaf(so[w][tr][e0 + k], f, o[k]);
    }
    const int sr = u.tile * kRowTile + tr;
    if (sr >= set.rows * a.group) return;
    const int row = set.first + sr / a.group, head = kvh * a.group + sr % a.group;
    if (direct) {
        const float inv = L != 0.0f ? 1.0f / L : 0.0f;
        float* dst = a.out + (size_t)row * a.out_ld + (size_t)head * HD + e0;
#pragma unroll
        for (int k = 0; k < NJ; k++) dst[k] = o[k] * inv;
    } else {
        const size_t at = part_at(tr, row, head);
        float* dst = a.po + at * HD + e0;
#pragma unroll
        for (int k = 0; k < NJ; k++) dst[k] = o[k];
        // (NaN scores alone leave the reference at -inf: 0 marks the part as there)
        if ((tid & 15) == 0) a.pml[at] = make_float2(M == -INFINITY && L != 0.0f ? 0.0f : M, L);
    }
}

// Many rows over the same pages (prompts, a prefix under a batch) of an f16 or
// bf16 cache: eight wavefronts of a row tile each share tiles of K and V in
// LDS, which LDS DMA brings in while the tile before is computed.  In LDS a row's
// pieces are permuted by the row (piece ^ row), so that the rows that an operand
// reads at one piece lie in different banks (no conflicts counted).  Bound by
// matrix and vector instructions, which hardly overlap: four prompts of 7781
// tokens, 32 heads on 8, f16, hd 64: 256 us, 370 TFLOP/s of the 4 hd per pair
// that a user sees, twice that in the two parts; counters: matrix cores 39% of
// the time, vector instructions 49%, clock 2.05 GHz.  Measured and dropped: two
// row tiles a wavefront (309 us), 4 wavefronts (281), 128 positions a tile
// (262); at hd 128, 12 and 16 wavefronts spill (bf16 326 us -> 412 and 699).
constexpr int kTileWaves = 8, kTileRows = kTileWaves * kRowTile;
// Of 4 rows by 16 columns of halfwords, of which the 16 lanes of a row of the
// wavefront point to four halfwords each, lane c gets column c.
__device__ __forceinline__ u2 load_transposed(const char* p) {
    typedef short s4 __attribute__((ext_vector_type(4)));
    return __builtin_bit_cast(u2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4*)p));
}
// 16 bytes per lane from `src` to LDS at `dst` + 16 lane
__device__ __forceinline__ void load_to_lds(const char* src, char* dst) { __builtin_amdgcn_global_load_lds(src, dst, 16, 0, 0); }
template <typename C, int HD>
__global__ __launch_bounds__(64 * kTileWaves, HD == 128 ? 2 : 4) void k_paged_attn_tile(PagedAttn a, int prefix) {
    using R = Tile<C, HD, true>;
    constexpr int NT = R::NT, NK = R::NK, NJ = R::NJ, STEP = R::STEP;
    constexpr int RB = HD * (int)sizeof(C), PIECES = RB / 16;          // bytes and pieces of a row
    constexpr int POS = 64;                                            // positions of a tile
    constexpr int PER = PIECES >= 16 ? 1 : 16 / PIECES;                // rows of 256 bytes
    constexpr int SWZ = PIECES >= 16 ? 15 : PIECES - 1;
    constexpr int VSWZ = PIECES / 2 - 1;                               // values: 32 bytes of a row, so that eight rows differ
    constexpr int ROWS = kTileRows;
    __shared__ __align__(16) char lds[2][2][POS * RB];                 // [buffer][keys, values]

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int c = lane & 15, g = lane >> 4;
    const int kvh = blockIdx.x % a.p.n_kv, split = blockIdx.y;
    const int slot = (int)(gridDim.x / a.p.n_kv) - 1 - (int)(blockIdx.x / a.p.n_kv);    // a sequence's last rows, the longest, first
    RowSet set;
    int tile;
    if (prefix) {
        set = prefix_set(a);
        tile = slot;
    } else if (!tile_of_slot(a, slot, __builtin_ctz(ROWS), &set, &tile) || row_kernel_takes(set.rows, a.group)) {
        return;
    }
    R r;
    int wave_most, least;
    r.place(a, set, tile * ROWS + wave * kRowTile, kvh, c);
    r.reach(a, set, &wave_most, &least);
    // the longest row of the workgroup
    int* reach = reinterpret_cast<int*>(lds);
    if (lane == 0) reach[wave] = wave_most;
    __syncthreads();
    int all = reach[0];
#pragma unroll
    for (int w = 1; w < kTileWaves; w++) all = max(all, reach[w]);
    __syncthreads();
    int lo, hi;
    split_range(a, split, all, &lo, &hi);
    if (lo >= hi && !a.direct) {
        if (r.live && g == 0) a.pml[part_of(a, r.row, r.head, split)] = make_float2(-INFINITY, 0.0f);
        return;
    }
    r.load_q(a, g);

    const int slots = (1 << a.p.page_shift) - 1;
    const int tiles = (hi - lo + POS - 1) / POS;
    // Pages of the next 64 16-position stretches, one per lane; of the tile being computed and the one on its way.
    const auto pages_from = [&](int at) { return at < hi ? paged_page(set.pages[at >> a.p.page_shift], a.p.n_pages) : -1; };
    constexpr int S = POS / 16;
    int page_reg = pages_from(lo + 16 * lane), next_reg = page_reg;
    // Brings a tile's keys and values into a buffer: RB bytes per position, 1024 per instruction.
    const int prow = lane / PIECES, piece = lane % PIECES;
    constexpr int PI = 1024 / RB, N = POS / PI;                // positions per instruction, instructions
    const auto fetch = [&](int t, int reg, int buffer) {
#pragma unroll
        for (int n = 0; n < (2 * N + kTileWaves - 1) / kTileWaves; n++) {
            const int i = wave + kTileWaves * n;
            if (i < 2 * N) {
                const bool key = i < N;
                const int row = (key ? i : i - N) * PI;        // of the tile, the instruction's first
                const int page = __builtin_amdgcn_readlane(reg, (t % (64 / S)) * S + row / 16);
                const char* src = static_cast<const char*>(key ? a.p.keys : a.p.values) +
                                  paged_offset(a.p, max(page, 0), kvh, (lo + POS * t + row) & slots) * sizeof(C);
                const int r16 = (row + prow) & 15;
                const uint32_t at = prow * RB + 16 * (piece ^ (key ? (r16 / PER) & SWZ : 2 * ((r16 / PER) & VSWZ)));
                load_to_lds(src + at, &lds[buffer][key ? 0 : 1][row * RB]);
            }
        }
    };
    // where a lane's pieces of a key, and of its values, stand in a stretch of
    // 16 positions (the permutations repeat)
    static_assert((16 / PER) % (SWZ + 1) == 0 && (16 / PER) % (VSWZ + 1) == 0, "16 positions hold whole permutations");
    int k_at[NK], v_at[NJ];
#pragma unroll
    for (int i = 0; i < NK; i++) k_at[i] = c * RB + 16 * ((4 * i + g) ^ ((c / PER) & SWZ));
    // (of the 4 rows by 16 dimensions that 16 lanes transpose, lane c brings row c / 4, dimensions 4 (c % 4) on)
    const int v_row = 4 * g + c / 4, v_swz = (v_row / PER) & VSWZ;
#pragma unroll
    for (int j = 0; j < NJ; j++) v_at[j] = v_row * RB + 32 * (j ^ v_swz) + 8 * (c & 3);
    fetch(0, page_reg, 0);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    lds_barrier();
    for (int t = 0; t < tiles; t++) {
        const int buffer = t & 1;
        if (t + 1 < tiles) {
            next_reg = (t + 1) % (64 / S) ? page_reg : pages_from(lo + POS * (t + 1) + 16 * lane);
            fetch(t + 1, next_reg, buffer ^ 1);
        }
        const char* kt = lds[buffer][0];
        const char* vt = lds[buffer][1];
        // a whole tile of positions per row tile at once: independent chains of
        // products, one look at the reference
        constexpr int NS = POS / STEP;
        const int p0 = lo + POS * t;
        if (p0 < min(wave_most, hi)) {
            int page[NS][NT];
            bool edge = p0 + POS > min(least, hi);
#pragma unroll
            for (int st = 0; st < NS; st++)
#pragma unroll
                for (int u = 0; u < NT; u++) {
                    page[st][u] = __builtin_amdgcn_readlane(page_reg, (t % (64 / S)) * S + st * NT + u);
                    edge = edge || page[st][u] < 0;
                }
            float s[NS * NT][4];
#pragma unroll
            for (int st = 0; st < NS; st++) {
                u4 kc[NT][NK];
#pragma unroll
                for (int u = 0; u < NT; u++)
#pragma unroll
                    for (int i = 0; i < NK; i++) kc[u][i] = *reinterpret_cast<const u4*>(kt + (STEP * st + 16 * u) * RB + k_at[i]);
                r.scores(kc, s + NT * st);
                if (edge) r.mask(s + NT * st, p0 + STEP * st, hi, page[st], g);
            }
            r.template weigh<NS * NT>(s);
#pragma unroll
            for (int st = 0; st < NS; st++) {
                const int ps = p0 + STEP * st;
                u4 vf[NJ];
#pragma unroll
                for (int j = 0; j < NJ; j++)
#pragma unroll
                    for (int u = 0; u < NT; u++) {
                        const u2 x = load_transposed(vt + (STEP * st + 16 * u) * RB + v_at[j]);
                        vf[j][2 * u] = x[0];
                        vf[j][2 * u + 1] = x[1];
                    }
                const bool odd = edge && clear_operands<C, HD>(vf, ps, hi, ps + STEP > least, page[st], g);
                r.add(s + NT * st, vf);
                if (odd) r.add_odd(a, s + NT * st, ps, hi, page[st], kvh, c, g);
            }
        }
        page_reg = next_reg;
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");       // the next tile is there
        lds_barrier();
    }

    const float L = r.sum();
    if (!r.live) return;
    float f = 1.0f;
    float* dst;
    if (a.direct) {
        f = L != 0.0f ? 1.0f / L : 0.0f;
        dst = a.out + (size_t)r.row * a.out_ld + (size_t)r.head * HD;
    } else {
        const size_t at = part_of(a, r.row, r.head, split);
        dst = a.po + at * HD;
        if (g == 0) a.pml[at] = make_float2(r.m == -INFINITY && L != 0.0f ? 0.0f : r.m, L);
    }
#pragma unroll
    for (int j = 0; j < NJ; j++) {
        const vf4 x = r.acc[j] * f;
        *reinterpret_cast<f4u*>(dst + R::dim(0, j, g)) = f4u{x[0], x[1], x[2], x[3]};
    }
}

// Where one list of partial results begins and how far its entries are apart.
struct Parts {
    const float* po; const float2* pml;
    size_t first; int step, n;
};

// Joins the partial results of a row, a wavefront per head (every fourth of
// `heads` heads): weights 2^(m - max), HD / 64 (or one) dimensions per lane.
// Bound by its round trips (lengths, weights, values): 4 to 7 us; a workgroup
// per head with two barriers took 12 us for 96 rows of 32 heads, now 6.
// `per_seq`: rows of every sequence that the row kernel took (that many of
// each are looked at); 0: all rows.  Their own parts stand at `rows`, those
// of the tile kernel (tile_parts, 0: it wrote `out`) and over the prefix at a.po.
template <int HD>
__global__ __launch_bounds__(256) void k_paged_attn_join(PagedAttn a, int heads, int per_seq, const float* rows_po, const float2* rows_pml,
                                                         int tile_parts, int prefix_parts) {
    constexpr int E = HD < 64 ? 1 : HD / 64;
    const int groups = (a.p.n_heads + heads - 1) / heads;
    const int at = blockIdx.x / groups, head0 = (blockIdx.x % groups) * heads;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int s = per_seq ? at / per_seq : paged_seq_of_row(a.p, at);
    if (s < 0) return;
    int first, end;
    paged_rows(a.p, s, &first, &end);
    const int row = per_seq ? first + at % per_seq : at;
    if (row < first || row >= end) return;
    const bool by_rows = !a.both || row_kernel_takes(end - first, a.group);
    int4 u = make_int4(0, tile_parts, 0, 0);
    if (by_rows) {
        if (!a.joined) return;                             // not split: written by its kernel
        u = a.wanted ? a.units[s] : make_int4(a.p.row_start ? first_slot(a, s, kRowTileLog2) : s * a.per, 1, 0, 0);
    }
    if (prefix_parts == 0 && (by_rows ? u.y == 1 : u.y == 0)) return;
    for (int head = head0 + wave; head < min(head0 + heads, a.p.n_heads); head += 4) {
        Parts own{a.po, a.pml, ((size_t)row * a.p.n_heads + head) * a.parts, 1, tile_parts};
        if (by_rows) {
            const int k = (row - first) * a.group + head % a.group, tile = k / kRowTile;
            const int64_t unit = (int64_t)u.x + (int64_t)tile * u.y;
            if (u.x < 0 || u.y < 1 || unit + u.y > a.max_units) return;    // (starts that do not ascend)
            own = Parts{rows_po, rows_pml, ((size_t)unit * a.p.n_kv + head / a.group) * kRowTile + k % kRowTile, a.p.n_kv * kRowTile, u.y};
        }
        const Parts pre{a.po, a.pml, ((size_t)row * a.p.n_heads + head) * a.parts + tile_parts, 1, prefix_parts};
        const int parts = own.n + pre.n;
        const auto index = [&](int i) { return i < own.n ? own.first + (size_t)i * own.step : pre.first + (size_t)(i - own.n); };
        const auto ml = [&](int i) { return i < parts ? (i < own.n ? own.pml : pre.pml)[index(i)] : make_float2(-INFINITY, 0.0f); };
        float2 v = ml(lane);
        float M = v.x;
        for (int i = 64 + lane; i < parts; i += 64) M = fmaxf(M, ml(i).x);
        M = wave_max(M);
        // 64 parts' weights at a time, one per lane; 16 parts' values in flight
        // (a part that is not there has weight 0, its values are not looked at)
        float L = 0.0f, o[E] = {};
        for (int b = 0; b < parts; b += 64) {
            if (b) v = ml(b + lane);
            const float w = v.x == -INFINITY ? 0.0f : v.x == M ? 1.0f : __builtin_amdgcn_exp2f(v.x - M);
            L += w == 0.0f ? 0.0f : w * v.y;
            const int n = min(64, parts - b);
            for (int j = 0; j < n; j += 16) {
                float x[16][E];
#pragma unroll
                for (int k = 0; k < 16; k++) {
                    const int i = b + min(j + k, n - 1);
                    const float* po = (i < own.n ? own.po : pre.po) + index(i) * HD;
#pragma unroll
                    for (int e = 0; e < E; e++) x[k][e] = po[E * min(lane, HD / E - 1) + e];
                }
#pragma unroll
                for (int k = 0; k < 16; k++) {
                    const float f = j + k < n ? lane_value(w, j + k) : 0.0f;
#pragma unroll
                    for (int e = 0; e < E; e++)
                        if (f != 0.0f) o[e] = fmaf(x[k][e], f, o[e]);
                }
            }
        }
        L = wave_sum(L);
        float* dst = a.out + (size_t)row * a.out_ld + (size_t)head * HD;
#pragma unroll
        for (int e = 0; e < E; e++)
            if (HD >= 64 || lane < HD) dst[E * lane + e] = L != 0.0f ? o[e] / L : 0.0f;
    }
}

// ------------------------------------------------------------------- host

namespace {

// How a call is split, from what the host knows of it.
struct Launch {
    int tiles = 0, splits = 1, chunk = 0;
};
struct AttnPlan {
    int per = 1, wanted = 0, max_units = 0;          // row kernel, own pages (PagedAttn)
    float finer = 0.0f;
    bool split = false, join_rows = false, both = false;
    int per_seq = 0;                                 // joining only what the row kernel took: rows of a sequence
    int tile_groups = 0;                             // tile kernel, own pages (not split): row tiles
    Launch prefix;
    bool prefix_by_tile = false;
    int tile_parts = 0;
    size_t row_units = 0, all_units = 0, bytes = 0;
};

// Own positions up to which a tile's are not split (one kernel less): of few
// tiles, of many.  One decoded row, 32 heads on 8, f16, hd 64, unsplit | split, in
// us: 300 positions 7.0 | 8.9, 600 8.3 | 8.9, 1000 10.3 | 9.2, 2000 15.5 | 9.0.
// Many (kManyTiles tiles of all kv heads), f32 prompts of hd 64: 1000 tokens 57.4 |
// 64.8, 1500 106 | 114, 3000 365 | 373; 8 turns of 60 tokens at 3000 positions, f16
// hd 64 87.2 | 76.8, bf16 hd 128 118 | 122.  Near kManyTiles: prompts of 130
// tokens (264 tiles) at 1000 positions, f32, 25.1 | 32.2, of 300 (608) 32.4 | 36.6, f16
// 20.2 | 24.3.
constexpr int kUnsplit = 640, kUnsplitMany = 2048, kManyTiles = 512;
// Tiles of all kv heads, one row per sequence, from which on a tile is split above
// the mean length, not above half of it.  Sequences of 100 .. 3000, bf16 hd 128, in us,
// mean | half: 140 (1120 tiles) 108 | 111, 240 173 | 183, 300 218 | 235, 500 373 |
// 412; of 100 .. 8000, f16 hd 64: 140 113 | 110, 240 171 | 172, 300 216 | 219, 500
// 363 | 378.
constexpr int kEnough = 2048;
// Positions of a part at least.  One decoded row, f16 hd 64, in us, 64 | 128 | 256: 700
// positions 10.3 | 10.3 | 11.0, 1000 10.3 | 10.6 | 11.3, 2000 11.6 | 10.3 | 11.0, 4000
// 14.8 | 11.7 | 11.2; bf16 hd 128: 1000 12.0 | 12.6 | 13.7, 4000 18.2 | 15.0 | 15.2; four
// rows under a prefix of 1500 15.3 | 14.0 | 15.0.
constexpr int kLeastChunk = 128;
// The tile kernel from as many workgroups of rows on (f16 and bf16 caches; f32's
// matrix instructions take so long that K and V need not be shared).  One prompt
// over itself, 32 heads on 8, in us, row kernel | tile kernel:
//   tokens            400            500            640            800           1280
//   workgroups        104            128            160            200            320
//   f16 hd 64   13.1 | 19.4    15.3 | 20.9    28.1 | 26.9    35.2 | 30.0    63.3 | 44.6
//   bf16 hd 128 26.0 | 32.5    27.5 | 35.7    46.7 | 47.3    58.7 | 54.1     104 | 79.0
// f32, 1280 tokens: 9 heads on 3, hd 64, 42.8 | 110; 32 on 8, hd 128, 187 | 214.
constexpr int kTileKernelGroups = 160;
// The tile kernel for a prefix from as many stacked rows of all kv heads times
// prefix positions on.  Decoded rows, 32 heads on 8, whole call in us, row
// kernel | tile kernel:
//   sequences x prefix    32 x 2000      32 x 6000      96 x 2000      96 x 6000
//   product (2^20)              2.0            5.9            5.9           17.6
//   f16 hd 64           19.9 | 22.5    26.8 | 31.5    34.4 | 37.1    56.6 | 41.4
//   bf16 hd 128         27.7 | 33.4    36.5 | 35.2    52.0 | 48.9    88.7 | 66.6
constexpr int64_t kPrefixByTile = 8 << 20;

// (units: where each sequence's begin)
size_t bytes_of(const PagedArgs& p, size_t row_units, size_t all_units) {
    const size_t bytes = (row_units + all_units) * (p.hd + 2) * sizeof(float);
    return bytes ? ((bytes + 15) & ~(size_t)15) + (size_t)p.n_seqs * sizeof(int4) : 0;
}

// Workgroups of the tile kernel that run at once (their registers).
int tile_resident(const PagedArgs& p) { return p.hd == 128 ? 256 : 512; }

AttnPlan plan_attention(const PagedArgs& p, int dtype, uint32_t max_len) {
    AttnPlan r;
    const int group = p.n_heads / p.n_kv, R = kTileRows;
    const int64_t cap = paged_capacity(p), stacked = (int64_t)p.n_rows * group;
    const int64_t longest = max_len && max_len < cap ? max_len : cap;
    const int own = (int)std::max<int64_t>(longest - p.prefix_len, 0);
    // splits the positions of `tiles` tiles so that `wanted` workgroups have work
    const auto split = [&](Launch* l, int64_t tiles, int positions, int wanted) {
        const int64_t want = std::max<int64_t>(wanted / std::max<int64_t>(tiles * p.n_kv, 1), 1);
        l->splits = (int)std::clamp<int64_t>(want, 1, std::max(1, (positions + kLeastChunk - 1) / kLeastChunk));
        l->chunk = ((positions + l->splits - 1) / l->splits + 63) & ~63;
        l->splits = std::max(1, (positions + l->chunk - 1) / std::max(l->chunk, 1));
    };
    r.both = p.row_start && dtype != YL_T_F32 && (stacked + R - 1) / R * p.n_kv >= kTileKernelGroups;
    r.per = (group + kRowTile - 1) / kRowTile;
    // tiles of the row kernel at most: slots of tile_of_slot, or fewer where the
    // tile kernel has the large sequences and the units are counted through (where
    // slots, most of them unused, are many: 8 prompts of 600 tokens beside 64 decoded rows at
    // 500, 20 slots a sequence, f16 hd 64, in us, search | count 91.8 | 79.1, 6 beside 30
    // 62.8 | 55.7; 2 beside 500, 2 slots a sequence, 165 | 191)
    const int64_t slots = stacked / kRowTile + p.n_seqs;
    const bool many = p.n_seqs > kDivided;
    r.split = !many && own > (p.row_start && !r.both && slots * p.n_kv >= kManyTiles ? kUnsplitMany : kUnsplit);
    const bool search = !r.split && (!r.both || many || slots <= 4 * (int64_t)p.n_seqs);
    const int64_t tiles = !p.row_start          ? (int64_t)p.n_seqs * r.per
                          : r.both && !search ? std::min<int64_t>((int64_t)p.n_seqs * (kRowKernelRows / kRowTile), slots)
                                              : slots;
    r.wanted = r.split ? std::max(1, 512 / p.n_kv) : p.row_start && !search ? 1 : 0;
    // One row per sequence: lengths differ, tiles of more than half the mean are
    // split (64 sequences of 100 .. 8000 139 -> 134 us; 128, hd 64, 98 against 102
    // for those above the mean), those above the mean where there are workgroups
    // enough (512 sequences 380 -> 373, of 100 .. 3000 232 -> 210).  Rows of
    // prompts: tiles of one length, which stay whole where there are many.
    r.finer = p.row_start ? 0.95f : tiles * p.n_kv >= kEnough ? 1.0f : 2.0f;
    r.max_units = (int)(tiles + std::max<int64_t>(r.wanted, r.split ? (int64_t)std::ceil(r.finer * (float)tiles) + 1 : 0));
    r.join_rows = r.split || p.prefix_len;
    if (r.both) r.tile_groups = (int)(stacked / R) + p.n_seqs;
    if (p.prefix_len) {
        r.prefix_by_tile = dtype != YL_T_F32 && stacked * p.n_kv * p.prefix_len >= kPrefixByTile;
        r.prefix.tiles = (int)((stacked + (r.prefix_by_tile ? R : kRowTile) - 1) / (r.prefix_by_tile ? R : kRowTile));
        split(&r.prefix, r.prefix.tiles, p.prefix_len, r.prefix_by_tile ? tile_resident(p) : 512);
    } else {
        r.prefix.splits = 0;
    }
    // partial results: of the row kernel, 16 rows for every unit and kv head;
    // of the others, for every row
    r.tile_parts = r.both && p.prefix_len ? 1 : 0;
    if (r.join_rows) r.row_units = (size_t)r.max_units * p.n_kv * kRowTile;
    r.all_units = (size_t)p.n_rows * p.n_heads * (r.tile_parts + r.prefix.splits);
    r.per_seq = r.both ? std::max(1, kRowKernelRows / group) : 0;
    if (r.all_units || (int64_t)p.n_seqs * r.per_seq >= p.n_rows) r.per_seq = 0;
    r.bytes = bytes_of(p, r.row_units, r.all_units);
    return r;
}

// What every call of no more sequences, rows, entries, positions and prefix
// takes: the largest of plan_attention's over them, or a little more.
size_t bytes_at_most(const PagedArgs& p, int dtype, uint32_t max_len) {
    const int group = p.n_heads / p.n_kv, R = kTileRows;
    const int64_t stacked = (int64_t)p.n_rows * group, entries = (int64_t)p.max_pages << p.page_shift;
    const int64_t own = max_len && max_len < entries ? max_len : entries;
    const bool tiled = dtype != YL_T_F32;
    const auto tiles_of = [&](int64_t rows, int64_t seqs) { return rows / kRowTile + seqs; };
    const auto finer = [](float f, int64_t tiles) { return (int64_t)std::ceil(f * (float)tiles) + 1; };
    int64_t units = 0;
    if (own > kUnsplit) {
        const int64_t seqs = std::min(p.n_seqs, kDivided), wanted = std::max(1, 512 / p.n_kv);
        // row_start: batches without the tile kernel have few stacked rows (of f32, all), and few
        // tiles while contexts are short; of the others, the row kernel has sequences of few rows
        int64_t tiles = tiles_of(tiled ? std::min<int64_t>(stacked, (int64_t)R * ((kTileKernelGroups - 1) / p.n_kv)) : stacked, seqs);
        if (own <= kUnsplitMany) tiles = std::min<int64_t>(tiles, (kManyTiles - 1) / p.n_kv);
        if (tiled) tiles = std::max(tiles, std::min(seqs * (kRowKernelRows / kRowTile), tiles_of(stacked, seqs)));
        units = tiles + std::max(wanted, finer(0.95f, tiles));
        // one row per sequence: twice the tiles' number again up to kEnough of all kv heads
        const int64_t single = std::min<int64_t>(seqs, p.n_rows) * ((group + kRowTile - 1) / kRowTile);
        const int64_t few = std::min<int64_t>(single, (kEnough - 1) / p.n_kv);
        units = std::max({units, single + std::max(wanted, finer(1.0f, single)), few + finer(2.0f, few)});
    }
    size_t all = 0;
    if (p.prefix_len) {
        units = std::max(units, tiles_of(stacked, p.n_seqs) + 1);
        // a part of the tile kernel, and the prefix's: more than one per row only where
        // the tiles of 16 or 128 rows are fewer than the workgroups wanted
        const int64_t heads = (int64_t)p.n_rows * p.n_heads, parts = (p.prefix_len + kLeastChunk - 1) / kLeastChunk;
        const int64_t wanted = tiled && heads * p.prefix_len >= kPrefixByTile ? (int64_t)tile_resident(p) * R : 512 * kRowTile;
        all = heads * (tiled && (stacked + R - 1) / R * p.n_kv >= kTileKernelGroups) + std::max(heads, std::min(heads * parts, wanted));
    }
    return bytes_of(p, (size_t)units * p.n_kv * kRowTile, all);
}

// The workspace that a call asks for.
size_t workspace_of(const PagedArgs& p, int dtype, uint32_t max_len, const AttnPlan& plan) {
    return std::max(plan.bytes, bytes_at_most(p, dtype, max_len));
}

template <typename C, int HD>
hipError_t launch_attn_hd(const PagedAttn& a, const dim3& grid, bool by_tile, bool prefix, hipStream_t s) {
    if constexpr (sizeof(C) == 2) {
        if (by_tile) {
            hipLaunchKernelGGL((k_paged_attn_tile<C, HD>), grid, dim3(64 * kTileWaves), 0, s, a, prefix);
            return hipGetLastError();
        }
    }
    hipLaunchKernelGGL((k_paged_attn_rows<C, HD>), grid, dim3(256), 0, s, a, prefix);
    return hipGetLastError();
}

template <typename C>
hipError_t launch_attn(const PagedAttn& a, const dim3& grid, bool by_tile, bool prefix, hipStream_t s) {
    return a.p.hd == 32 ? launch_attn_hd<C, 32>(a, grid, by_tile, prefix, s) : a.p.hd == 64 ? launch_attn_hd<C, 64>(a, grid, by_tile, prefix, s)
                                                                           : launch_attn_hd<C, 128>(a, grid, by_tile, prefix, s);
}

template <typename C>
hipError_t launch_all(PagedAttn a, const AttnPlan& plan, float* space, hipStream_t s) {
    const size_t units = plan.row_units + plan.all_units;
    float* const all_po = space + plan.row_units * a.p.hd;
    float2* const ml = reinterpret_cast<float2*>(space + units * a.p.hd);
    float2* const all_ml = ml + plan.row_units;
    a.both = plan.both;
    a.per = plan.per; a.wanted = plan.wanted; a.finer = plan.finer; a.max_units = plan.max_units;
    a.units = reinterpret_cast<int4*>(reinterpret_cast<char*>(space) + (plan.bytes - (size_t)a.p.n_seqs * sizeof(int4)));
    a.po = space; a.pml = ml;
    a.direct = !a.p.prefix_len;
    a.joined = plan.join_rows;
    a.chunk = plan.split ? kLeastChunk : 1 << 30;
    hipError_t e = launch_attn<C>(a, dim3((unsigned)plan.max_units * a.p.n_kv), false, false, s);
    a.po = all_po; a.pml = all_ml;
    a.parts = plan.tile_parts + plan.prefix.splits;
    if (e == hipSuccess && plan.both) {
        a.direct = !plan.tile_parts;
        a.splits = 1;
        e = launch_attn<C>(a, dim3((unsigned)plan.tile_groups * a.p.n_kv), true, false, s);
    }
    if (e == hipSuccess && a.p.prefix_len) {
        a.direct = 0;
        a.part0 = plan.tile_parts;
        a.splits = plan.prefix.splits; a.chunk = plan.prefix.chunk;
        e = launch_attn<C>(a, dim3((unsigned)plan.prefix.tiles * a.p.n_kv, plan.prefix.splits), plan.prefix_by_tile, true, s);
    }
    if (e != hipSuccess || !units) return e;    // (nothing was split)
    const int rows = plan.per_seq ? a.p.n_seqs * plan.per_seq : a.p.n_rows;
    const int heads = (int)std::clamp<int64_t>((int64_t)rows * a.p.n_heads / 4096, 4, std::max(4, a.p.n_heads));
    const dim3 grid((unsigned)rows * ((a.p.n_heads + heads - 1) / heads));
    auto join = a.p.hd == 32 ? k_paged_attn_join<32> : a.p.hd == 64 ? k_paged_attn_join<64> : k_paged_attn_join<128>;
    hipLaunchKernelGGL(join, grid, dim3(256), 0, s, a, heads, plan.per_seq, (const float*)space, (const float2*)ml,
                       plan.tile_parts, plan.prefix.splits);
    return hipGetLastError();
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
    return workspace_of(p, cache->dtype, batch->max_len, plan_attention(p, cache->dtype, batch->max_len));
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
    const AttnPlan plan = plan_attention(a.p, cache->dtype, batch->max_len);
    const size_t need = workspace_of(a.p, cache->dtype, batch->max_len, plan);
    if (need && (!workspace || (uintptr_t)workspace % 16)) return refuse("paged_attention: the workspace has to be there, 16-byte aligned");
    if (workspace_bytes < need) return refuse("paged_attention: the workspace is smaller than yl_paged_attention_workspace says", YL_ERR_RANGE);
    a.out = out; a.q = q; a.out_ld = out_ld; a.q_ld = q_ld;
    a.scale = frexpf(attn_scale * 1.4426950408889634f, &a.scale_exp);
    a.group = a.p.n_heads / a.p.n_kv;
    hipStream_t s = (hipStream_t)stream;
    float* space = static_cast<float*>(workspace);
    const hipError_t e = cache->dtype == YL_T_F32   ? launch_all<float>(a, plan, space, s)
                         : cache->dtype == YL_T_F16 ? launch_all<_Float16>(a, plan, space, s)
                                                    : launch_all<__bf16>(a, plan, space, s);
    if (e == hipSuccess) return YL_OK;
    set_error(std::string("paged_attention launch: ") + hipGetErrorString(e));
    return YL_ERR_HIP;
}

}  // extern "C"
