// yl_logprobs.hip -- log probabilities of given tokens, the entropy and the
// most probable alternatives of rows of logits.  No counterpart in the
// reference (sampler.rs holds one row of probabilities on the host).
//
//   lse = m + log Z, Z = sum exp(x - m);  log p_i = (x_i - m) - log Z
//   H = log Z - sum (x - m) exp(x - m) / Z     (both terms are >= 0)
// log Z is taken as log1p of Z - 1, summed without the maximum's own 1, so that
// a sharp row keeps the small rest.  Bound by reading the logits once: 700 rows
// of 128256 f32 64 us, 5.6 TB/s (one pass for the maximum, one for the sums and
// one per top entry: 1740 us); of bf16 64 us too, bound by the vector instructions;
// one row 11 us, two launches and three round trips.
#include <hip/hip_runtime.h>

#include <math.h>

#include <algorithm>

#include "../../include/yallma3.h"
#include "yl_device.h"
#include "yl_internal.h"

namespace yl {

constexpr int kTopMost = 32;
constexpr int kScoreThreads = 512;
constexpr int kCands = 1024;          // candidates of one selection

// A value's place in the order of the top list: NaN last, -0 with +0.
__device__ __forceinline__ uint32_t order_key(float x) {
    if (x != x) return 0u;
    const uint32_t b = __float_as_uint(x == 0.0f ? 0.0f : x);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
// Value and id in one order (falling: larger values, then smaller ids); never 0.
typedef unsigned long long u64;
__device__ __forceinline__ u64 id_key(float x, uint32_t i) { return ((u64)order_key(x) << 32) | (uint32_t)~i; }

// The value of a key (+0 for -0, NaN for any NaN).
__device__ __forceinline__ float key_value(u64 key) {
    const uint32_t k = (uint32_t)(key >> 32);
    return k == 0u ? NAN : __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k);
}

__device__ __forceinline__ float wave_sum(float v) {     // every lane active; the same order on every run
    v += dpp_mov<0xB1>(v);
    v += dpp_mov<0x4E>(v);
    v += dpp_mov<0x141>(v);
    v += dpp_mov<0x140>(v);
    return (lane_value(v, 0) + lane_value(v, 16)) + (lane_value(v, 32) + lane_value(v, 48));
}
__device__ __forceinline__ u64 wave_max64(u64 k) {
    for (int off = 32; off > 0; off >>= 1) {
        const u64 o = __shfl_xor(k, off, 64);
        if (o > k) k = o;
    }
    return k;
}

// e^d for d <= 0 (NaN of NaN, 0 from -200 on: *d is raised to it).  exp2 is right
// to an ulp, but its argument, d log2(e), is rounded, which at d = -30 would be 11
// ulp of the result: e^d = 2^t e^(d - t log(2)), whose second factor is
// 1 + (d - t log(2)) to 2^-39.
__device__ __forceinline__ float exp_below(float* d) {
    *d = __builtin_elementwise_maximum(*d, -200.0f);       // (keeps NaN)
    const float t = *d * 1.4426950408889634f, p = __builtin_amdgcn_exp2f(t);
    return fmaf(p, fmaf(t, -0.6931471805599453f, *d), p);
}

// A stretch of a row: its maximum, the sum of exp(x - m) over all but one
// holder of the maximum (whose 1 would hide the small ones), and the sum of
// (x - m) exp(x - m).  m = -inf with rest 0: nothing probable.
struct Stretch { float m, rest, t; };

__device__ __forceinline__ Stretch stretch_of(float m, float z, float t, int holders) {
    if (m == -INFINITY) return Stretch{m, z != z ? z : 0.0f, 0.0f};
    return Stretch{m, m == INFINITY ? NAN : z + (float)(holders - 1), t};
}
// Adds stretch b at the common maximum m; holder: whose maximum's 1 is left out.
__device__ __forceinline__ void add_stretch(const Stretch& b, float m, bool holder, float* rest, float* t) {
    if (b.m == -INFINITY) { *rest += b.rest; return; }         // (0, or NaN)
    float d = b.m - m;
    const float all = b.rest + 1.0f;
    if (holder) { *rest += b.rest; *t += b.t; return; }
    const float f = exp_below(&d);
    if (f == 0.0f && all == all) return;
    *rest = fmaf(all, f, *rest);
    *t = fmaf(f, fmaf(d, all, b.t), *t);
}

// The results of a row from its whole stretch.
struct RowScore {
    float m, lz, rest, t;
    bool none;
    __device__ explicit RowScore(const Stretch& s) : m(s.m), rest(s.rest), t(s.t), none(s.m == -INFINITY && s.rest == 0.0f) { lz = log1pf(s.rest); }
    __device__ float logprob(float x) const { return none ? -INFINITY : rest != rest ? rest : (x - m) - lz; }
    __device__ float entropy() const { return none ? 0.0f : rest != rest ? rest : lz - t / (1.0f + rest); }
};

// The `top` largest of n (<= kCands) distinct keys, by counting for each how
// many are larger: put(rank, key).  key[n .. n + 7] are 0.
template <typename Put>
__device__ __forceinline__ void rank_keys(const u64* key, int n, int top, int tid, int threads, Put put) {
    typedef u64 u64x2 __attribute__((ext_vector_type(2)));
    for (int i = tid; i < n; i += threads) {
        const u64 k = key[i];
        int r = 0;
        for (int j = 0; j < n; j += 8) {     // (eight keys in flight: one at a time, a read's latency each)
            u64x2 o[4];
#pragma unroll
            for (int e = 0; e < 4; e++) o[e] = *reinterpret_cast<const u64x2*>(key + j + 2 * e);
#pragma unroll
            for (int e = 0; e < 4; e++) r += (o[e].x > k) + (o[e].y > k);
        }
        if (k && r < top) put(r, k);
    }
}

// One workgroup per (stretch, row): the stretch's values stay in registers
// (8 V per thread), read once.  Sums: per thread, then over the workgroup; only
// the wavefronts that hold the maximum look for its holders.
// Top: of 64 groups of threads (one lane of each wavefront), the top-th largest
// group maximum has `top` values at or above it and so bounds the stretch's top
// values from below; the few values at or above the bound (some 25 of 4096 random
// ones at top 20) are ranked by counting.  Where equal values make them more
// than kCands, the entries are found one by one from memory (nothing but equal
// values in 700 rows of 128256, top 20: 1.07 ms; from the registers 0.56, which
// spills and costs every row a third).  Values of -inf and NaN are
// looked for by id, where the others do not fill the list.
template <typename T, int V>
__global__ __launch_bounds__(kScoreThreads, 6) void k_score(const T* __restrict__ x, size_t vocab, size_t ld, const uint32_t* tokens,
                                                            float* logprob, float* entropy, int top, uint32_t* top_ids,
                                                            float* top_logprobs, float4* part, u64* cand) {
    constexpr int W = 16 / (int)sizeof(T), N = 8 * V, G = N / W, NW = kScoreThreads / 64;
    typedef T vec __attribute__((ext_vector_type(W), aligned(sizeof(T))));
    __shared__ float gm[NW][64], rm[NW], rz[NW], rt[NW], least_sh;
    __shared__ int rc[NW];
    __shared__ __align__(16) u64 key[kCands + 8];
    __shared__ u64 rk[NW];
    __shared__ int count;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const size_t row = blockIdx.y, seg = blockIdx.x, base = seg * (size_t)(kScoreThreads * N);
    const T* __restrict__ xr = x + row * ld;
    const int n = (int)min((size_t)(kScoreThreads * N), vocab - base);
    float v[N];
#pragma unroll
    for (int k = 0; k < G; k++) {
        const int at = W * (tid + k * kScoreThreads);
        if (at + W <= n) {
            const vec c = *reinterpret_cast<const vec*>(xr + base + at);
#pragma unroll
            for (int e = 0; e < W; e++) v[W * k + e] = (float)c[e];
        } else {
#pragma unroll
            for (int e = 0; e < W; e++) v[W * k + e] = at + e < n ? (float)xr[base + at + e] : -INFINITY;
        }
    }
    float mx = v[0];
#pragma unroll
    for (int k = 1; k < N; k++) mx = fmaxf(mx, v[k]);
    mx = fmaxf(mx, -INFINITY);                           // (all NaN: nothing)
    float m = wave_max(mx);
    if (lane == 0) rm[wave] = m;
    if (top) gm[wave][lane] = mx;
    __syncthreads();
    if (top && wave == 0) {
        float g = gm[0][lane];
#pragma unroll
        for (int w = 1; w < NW; w++) g = fmaxf(g, gm[w][lane]);
        // the top-th largest, from its upper 20 bits on (a bound may be lower)
        const uint32_t mine = order_key(g);
        uint32_t b = 0;
        for (int bit = 31; bit >= 12; bit--) {
            const uint32_t c = b | (1u << bit);
            if (__builtin_popcountll(__ballot(mine >= c)) >= top) b = c;
        }
        if (lane == 0) {
            least_sh = b <= order_key(-INFINITY) ? -INFINITY : key_value((u64)b << 32);
            count = 0;
        }
    }
    m = rm[0];
#pragma unroll
    for (int w = 1; w < NW; w++) m = fmaxf(m, rm[w]);
    const float ms = m == -INFINITY ? 0.0f : m;
    float z = 0.0f, t = 0.0f;
    int holders = 0;
    // (-inf: weight 0 times the least difference; NaN stays NaN)
    if (__ballot(mx == m)) {
        int mine = 0;
#pragma unroll
        for (int k = 0; k < N; k++) {
            float d = v[k] - ms;
            const bool holds = d >= 0.0f;
            const float x = exp_below(&d), e = holds ? 0.0f : x;
            mine += holds;
            z += e;
            t = fmaf(d, e, t);
        }
        for (u64 left = __ballot(mine > 0); left; left &= left - 1) holders += __builtin_amdgcn_readlane(mine, __builtin_ctzll(left));
    } else {
#pragma unroll
        for (int k = 0; k < N; k++) {
            float d = v[k] - ms;
            const float e = exp_below(&d);
            z += e;
            t = fmaf(d, e, t);
        }
    }
    z = wave_sum(z);
    t = wave_sum(t);
    if (lane == 0) { rz[wave] = z; rt[wave] = t; rc[wave] = holders; }
    __syncthreads();
    z = t = 0.0f;
    holders = 0;
#pragma unroll
    for (int w = 0; w < NW; w++) { z += rz[w]; t += rt[w]; holders += rc[w]; }
    const Stretch st = stretch_of(m, z, t, holders);
    const bool whole = gridDim.x == 1;
    const size_t at = row * gridDim.x + seg;
    const RowScore score(st);
    if (tid == 0) {
        if (!whole) {
            part[at] = make_float4(st.m, st.rest, st.t, 0.0f);
        } else {
            if (logprob)
                logprob[row] = tokens[row] < vocab          ? score.logprob((float)xr[tokens[row]])
                               : score.rest != score.rest ? score.rest
                                                          : -INFINITY;
            if (entropy) entropy[row] = score.entropy();
        }
    }
    if (!top) return;
    const float least = least_sh;
    if (mx >= least && mx > -INFINITY) {
#pragma unroll
        for (int k = 0; k < N; k++) {
            const int i = W * (tid + (k / W) * kScoreThreads) + k % W;
            if (v[k] >= least && v[k] > -INFINITY) {         // (what is past n is -inf)
                const int c = atomicAdd(&count, 1);
                if (c < kCands) key[c] = id_key(v[k], (uint32_t)(base + i));
            }
        }
    }
    __syncthreads();
    const auto put = [&](int r, u64 k) {
        if (!whole) {
            cand[at * top + r] = k;
        } else {
            top_ids[row * top + r] = ~(uint32_t)k;
            top_logprobs[row * top + r] = score.logprob(key_value(k));
        }
    };
    const int found = count;
    if (found <= kCands) {
        if (tid < 8) key[found + tid] = 0;
        __syncthreads();
        rank_keys(key, found, top, tid, kScoreThreads, put);
        // Fewer than asked for (a choice of few tokens): then the ids of -inf
        // from the lowest on, then those of NaN, 64 values at a time.
        int filled = found;
        const int wanted = min(top, n);
        if (wave == 0) {
            for (int pass = 0; pass < 2 && filled < wanted; pass++)
                for (int i0 = 0; i0 < n && filled < wanted; i0 += 64) {
                    const float x0 = i0 + lane < n ? (float)xr[base + i0 + lane] : 0.0f;
                    const bool take = pass ? x0 != x0 : x0 == -INFINITY;
                    const u64 all = __ballot(take);
                    const int r = filled + __builtin_popcountll(all & ((1ull << lane) - 1));
                    if (take && r < wanted) put(r, id_key(x0, (uint32_t)(base + i0 + lane)));
                    filled += __builtin_popcountll(all);
                }
        }
        if (!whole)
            for (int r = wanted + tid; r < top; r += kScoreThreads) cand[at * top + r] = 0;
        return;
    }
    u64 last = ~0ull;
    for (int r = 0; r < top; r++) {
        u64 best = 0;
#pragma unroll 2
        for (int k = 0; k < G; k++) {
            const int i = W * (tid + k * kScoreThreads);
            if (i >= n) break;
            vec x;
            if (i + W <= n) x = *reinterpret_cast<const vec*>(xr + base + i);
            else
                for (int e = 0; e < W; e++) x[e] = xr[base + min(i + e, n - 1)];
#pragma unroll
            for (int e = 0; e < W; e++) {
                const u64 c = id_key((float)x[e], (uint32_t)(base + min(i + e, n - 1)));
                if (c < last && c > best) best = c;
            }
        }
        best = wave_max64(best);
        __syncthreads();
        if (lane == 0) rk[wave] = best;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < NW; w++)
            if (rk[w] > best) best = rk[w];
        last = best;
        if (tid == 0) put(r, best);
    }
}

// One workgroup per row: the stretches' sums at the common maximum, and the
// top keys of their lists.
template <typename T>
__global__ __launch_bounds__(256) void k_score_join(const T* __restrict__ x, size_t vocab, size_t ld, int segs, const uint32_t* tokens,
                                                    float* logprob, float* entropy, int top, uint32_t* top_ids,
                                                    float* top_logprobs, const float4* part, const u64* cand) {
    __shared__ float rm[4], rz[4], rt[4];
    __shared__ int rh[4];
    __shared__ __align__(16) u64 key[kCands + 8];
    __shared__ u64 rk[4];
    __shared__ int count;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const size_t row = blockIdx.x;
    const T* __restrict__ xr = x + row * ld;
    const float4* pr = part + row * segs;
    const u64* cr = cand + row * segs * top;
    const float chosen = logprob && tid == 0 && tokens[row] < vocab ? (float)xr[tokens[row]] : 0.0f;
    // Every list falls, so with j entries from each of the lists making up
    // `top`, the smallest of these j-th entries bounds the result from below.
    const bool few = segs * top <= kCands;
    u64 mine[kCands / 256], bound = ~0ull;
    if (top && few) {
        const int j = (top + segs - 1) / segs - 1;
#pragma unroll
        for (int k = 0; k < kCands / 256; k++) mine[k] = tid + 256 * k < segs * top ? cr[tid + 256 * k] : 0;
        for (int i = lane; i < segs; i += 64) bound = min(bound, cr[(size_t)i * top + j]);
        for (int off = 32; off > 0; off >>= 1) bound = min(bound, __shfl_xor(bound, off, 64));
        if (tid == 0) count = 0;
    }
    // the maximum, and the first stretch that holds it
    float m = -INFINITY;
    int at = 0x7fffffff;
    for (int i = tid; i < segs; i += 256) {
        const float v = pr[i].x;
        if (v > m || at == 0x7fffffff) { m = v; at = i; }
    }
    for (int off = 32; off > 0; off >>= 1) {
        const float om = __shfl_xor(m, off, 64);
        const int oa = __shfl_xor(at, off, 64);
        if (om > m || (om == m && oa < at)) { m = om; at = oa; }
    }
    if (lane == 0) { rm[wave] = m; rh[wave] = at; }
    __syncthreads();
    m = rm[0];
    at = rh[0];
#pragma unroll
    for (int w = 1; w < 4; w++)
        if (rm[w] > m || (rm[w] == m && rh[w] < at)) { m = rm[w]; at = rh[w]; }
    float rest = 0.0f, t = 0.0f;
    for (int i = tid; i < segs; i += 256) {
        const float4 p = pr[i];
        add_stretch(Stretch{p.x, p.y, p.z}, m, i == at, &rest, &t);
    }
    rest = wave_sum(rest);
    t = wave_sum(t);
    if (lane == 0) { rz[wave] = rest; rt[wave] = t; }
    if (top && few)
#pragma unroll
        for (int k = 0; k < kCands / 256; k++)
            if (mine[k] && mine[k] >= bound) key[atomicAdd(&count, 1)] = mine[k];
    __syncthreads();
    const RowScore score(Stretch{m, (rz[0] + rz[1]) + (rz[2] + rz[3]), (rt[0] + rt[1]) + (rt[2] + rt[3])});
    if (tid == 0) {
        if (logprob) logprob[row] = tokens[row] < vocab ? score.logprob(chosen) : score.rest != score.rest ? score.rest : -INFINITY;
        if (entropy) entropy[row] = score.entropy();
    }
    if (!top) return;
    const auto put = [&](int r, u64 k) {
        top_ids[row * top + r] = ~(uint32_t)k;
        top_logprobs[row * top + r] = score.logprob(key_value(k));
    };
    if (few) {
        if (tid < 8) key[count + tid] = 0;
        __syncthreads();
        rank_keys(key, count, top, tid, 256, put);
        return;
    }
    u64 last = ~0ull;
    for (int r = 0; r < top; r++) {
        u64 best = 0;
        for (size_t i = tid; i < (size_t)segs * top; i += 256) {
            const u64 c = cr[i];
            if (c < last && c > best) best = c;
        }
        best = wave_max64(best);
        __syncthreads();
        if (lane == 0) rk[wave] = best;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < 4; w++)
            if (rk[w] > best) best = rk[w];
        last = best;
        if (tid == 0) put(r, best);
    }
}

namespace {

// Values per thread of a stretch, 8 v, and the stretches of a row.
struct ScorePlan {
    int v = 2, segs = 1;
    size_t part_bytes = 0, bytes = 0;
};

// Stretches of 16384 values where at least one per CU is left of these, else
// of 8192 (more workgroups): rows of 128256, top 5, in us
//   rows     1      8     16     32     64    256
//   8192  10.8   11.2   11.8   13.9   17.4   34.7
//  16384  11.6   12.1   12.6   13.9   17.2   31.8
// (4096: 10.5, 11.4, 12.8, 16.4, 22.1, 52.8).  A row that one stretch of 16384
// holds needs no second kernel.
constexpr size_t kScoreEnough = 256;
ScorePlan plan_score(size_t rows, size_t vocab, uint32_t top) {
    ScorePlan p;
    const auto segs = [&](int v) { return (vocab + (size_t)kScoreThreads * 8 * v - 1) / ((size_t)kScoreThreads * 8 * v); };
    p.v = rows * segs(4) >= kScoreEnough || (segs(4) == 1 && segs(2) > 1) ? 4 : 2;
    p.segs = (int)segs(p.v);
    if (p.segs > 1) {
        p.part_bytes = rows * p.segs * sizeof(float4);
        p.bytes = p.part_bytes + rows * p.segs * top * sizeof(u64);
    }
    return p;
}

// What every call of no more rows, a vocabulary and a list no longer takes: fewer
// rows may be cut into the shorter stretches, fewer than 256 * 2 in all.
size_t score_bytes_at_most(size_t rows, size_t vocab, uint32_t top) {
    const auto segs = [&](int v) { return (vocab + (size_t)kScoreThreads * 8 * v - 1) / ((size_t)kScoreThreads * 8 * v); };
    if (segs(4) == 1) return 0;
    return std::max(rows * segs(4), std::min<size_t>(rows * segs(2), 2 * (kScoreEnough - 1))) * (sizeof(float4) + top * sizeof(u64));
}

struct ScoreArgs {
    const void* x; size_t rows, vocab, ld;
    const uint32_t* tokens; float* logprob; float* entropy;
    int top; uint32_t* ids; float* tlp; void* workspace;
};

template <typename T>
hipError_t launch_score(const ScoreArgs& a, const ScorePlan& p, hipStream_t s) {
    const T* x = static_cast<const T*>(a.x);
    float4* part = static_cast<float4*>(a.workspace);
    u64* cand = reinterpret_cast<u64*>(static_cast<char*>(a.workspace) + p.part_bytes);
    // (a grid has at most 65535 rows in y)
    for (size_t r = 0; r < a.rows; r += 65535) {
        const size_t n = std::min<size_t>(65535, a.rows - r), pr = r * p.segs;
        const auto at = [&](auto* base, size_t i) { return base ? base + i : base; };
        auto k = p.v == 2 ? k_score<T, 2> : k_score<T, 4>;
        hipLaunchKernelGGL(k, dim3(p.segs, (unsigned)n), dim3(kScoreThreads), 0, s, x + r * a.ld, a.vocab, a.ld, at(a.tokens, r),
                           at(a.logprob, r), at(a.entropy, r), a.top, at(a.ids, r * a.top), at(a.tlp, r * a.top), at(part, pr), at(cand, pr * a.top));
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess || p.segs == 1) {
            if (e != hipSuccess) return e;
            continue;
        }
        hipLaunchKernelGGL(k_score_join<T>, dim3((unsigned)n), dim3(256), 0, s, x + r * a.ld, a.vocab, a.ld, p.segs, at(a.tokens, r),
                           at(a.logprob, r), at(a.entropy, r), a.top, at(a.ids, r * a.top), at(a.tlp, r * a.top), at(part, pr), at(cand, pr * a.top));
        const hipError_t e2 = hipGetLastError();
        if (e2 != hipSuccess) return e2;
    }
    return hipSuccess;
}

}  // namespace
}  // namespace yl

using namespace yl;

extern "C" {

size_t yl_token_logprobs_workspace(size_t rows, size_t vocab, uint32_t top) {
    if (!rows || rows >= (1ull << 31) || !vocab || vocab >= (1ull << 31) || top > (uint32_t)kTopMost) return 0;
    return std::max(plan_score(rows, vocab, top).bytes, score_bytes_at_most(rows, vocab, top));
}

yl_status yl_token_logprobs(const void* logits, int32_t dtype, size_t rows, size_t vocab, size_t ld,
                            const uint32_t* tokens, float* logprob, float* entropy, uint32_t top, uint32_t* top_ids,
                            float* top_logprobs, void* workspace, size_t workspace_bytes, void* stream) {
    const auto refuse = [](const char* what, yl_status st = YL_ERR_ARG) { set_error(what); return st; };
    if (dtype != YL_T_F32 && dtype != YL_T_F16 && dtype != YL_T_BF16)
        return refuse("token_logprobs: logits are f32, f16 or bf16", YL_ERR_FORMAT);
    if (!vocab || vocab >= (1ull << 31) || ld < vocab) return refuse("token_logprobs: a vocabulary from 1 to below 2^31, rows at least as far apart");
    if (top > (uint32_t)kTopMost || top > vocab) return refuse("token_logprobs: top is at most 32 and at most the vocabulary");
    if (rows >= (1ull << 31)) return refuse("token_logprobs: fewer than 2^31 rows", YL_ERR_RANGE);
    if (rows == 0) return YL_OK;
    if (!logits || (uintptr_t)logits % (dtype == YL_T_F32 ? 4 : 2)) return refuse("token_logprobs: no logits, or not aligned to their type");
    if (!tokens != !logprob) return refuse("token_logprobs: tokens and logprob, or neither");
    if (top && (!top_ids || !top_logprobs)) return refuse("token_logprobs: top needs top_ids and top_logprobs");
    if (!logprob && !entropy && !top) return refuse("token_logprobs: nothing is asked for");
    const ScorePlan plan = plan_score(rows, vocab, top);
    const size_t need = std::max(plan.bytes, score_bytes_at_most(rows, vocab, top));
    if (need && (!workspace || (uintptr_t)workspace % 16)) return refuse("token_logprobs: the workspace has to be there, 16-byte aligned");
    if (workspace_bytes < need) return refuse("token_logprobs: the workspace is smaller than yl_token_logprobs_workspace says", YL_ERR_RANGE);
    const ScoreArgs a{logits, rows, vocab, ld, tokens, logprob, entropy, (int)top, top_ids, top_logprobs, workspace};
    hipStream_t s = (hipStream_t)stream;
    const hipError_t e = dtype == YL_T_F32 ? launch_score<float>(a, plan, s) : dtype == YL_T_F16 ? launch_score<_Float16>(a, plan, s)
                                                                                              : launch_score<__bf16>(a, plan, s);
    if (e == hipSuccess) return YL_OK;
    set_error(std::string("token_logprobs launch: ") + hipGetErrorString(e));
    return YL_ERR_HIP;
}

}  // extern "C"
