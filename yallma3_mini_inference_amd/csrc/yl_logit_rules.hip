// yl_logit_rules.hip -- what a row of logits is subject to before a token is
// chosen: penalties for tokens that are there already, biases, grammar masks.
// No counterpart in the reference.
//
// One pass over the logits.  A workgroup has a stretch of a row, eight logits per
// thread: it counts in LDS what of the row's tokens falls into its stretch (every
// workgroup of a row looks at all of them: they are few beside the logits and lie in
// L2), while its logits are on their way, and then changes each logit once.  Counts are
// whole numbers and of an id's biases the last in the list wins, so that the
// order of the LDS operations does not matter.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "../../include/yallma3.h"
#include "yl_device.h"
#include "yl_internal.h"

namespace yl {

namespace {

constexpr int kRuleThreads = 512, kRuleChunk = 8, kRuleStretch = kRuleThreads * kRuleChunk;

struct RuleArgs {
    const void* x; void* out;
    size_t vocab, ld, out_ld, row0;
    yl_logit_rules r;
};

// Entries [*begin, *end) of row `row` of a list of n entries.
__device__ __forceinline__ void entries_of(const uint32_t* start, uint32_t n, size_t row, uint32_t* begin, uint32_t* end) {
    const uint32_t b = start[row], e = start[row + 1];
    *end = min(e, n);
    *begin = min(b, *end);
}

}  // namespace

// Bound by memory where there are many rows: 256 of 128256 f32 logits 49 us, 5.3 TB/s in
// and out; one row 5 us: the launch and four round trips.  Entries of an id
// that nothing names are neither cleared nor read (with all of them 61 us); stores
// that L2 does not keep (60 -> 57 of two chunks per thread); two chunks per thread, which
// leaves two workgroups per CU beside their LDS, 60.
template <typename T>
__global__ __launch_bounds__(kRuleThreads) void k_logit_rules(RuleArgs a) {
    constexpr int W = kRuleThreads, N = kRuleChunk, S = kRuleStretch;
    typedef T Chunk __attribute__((ext_vector_type(N), aligned(sizeof(T))));
    __shared__ uint32_t count[S];                      // bit 31: among the row's tokens; below: how often after its prompt
    __shared__ uint32_t which[S];                      // 1 + place of the id's bias in the row's list
    __shared__ uint32_t named[S / 32];                 // a bit per id that a token or a bias names: only these have entries above
    const int tid = threadIdx.x;
    const size_t row = a.row0 + blockIdx.y, lo = (size_t)blockIdx.x * S, at = lo + (size_t)N * tid;
    const T* x = static_cast<const T*>(a.x) + row * a.ld;
    T* out = static_cast<T*>(a.out) + row * a.out_ld;
    uint32_t t0 = 0, t1 = 0, b0 = 0, b1 = 0;
    if (a.r.token_start) entries_of(a.r.token_start, a.r.n_tokens, row, &t0, &t1);
    if (a.r.bias_start) entries_of(a.r.bias_start, a.r.n_biases, row, &b0, &b1);
    Chunk v;
    if (at + N <= a.vocab) v = *reinterpret_cast<const Chunk*>(x + at);
    else
#pragma unroll
        for (int i = 0; i < N; i++) v[i] = at + i < a.vocab ? x[at + i] : (T)0.0f;
    // what of a list falls into the stretch, four entries per thread on their way
    const auto each = [&](const uint32_t* ids, uint32_t begin, uint32_t end, const auto& f) {
        for (uint32_t i = begin + tid; i < end; i += 4 * W) {
            size_t id[4];
#pragma unroll
            for (int k = 0; k < 4; k++) id[k] = ids[min(i + W * k, end - 1)];
#pragma unroll
            for (int k = 0; k < 4; k++)
                if (i + W * k < end && id[k] - lo < (size_t)S) f(i + W * k, (int)(id[k] - lo));       // (also below lo)
        }
    };
    // (more tokens than ids: all ids count as named, which spares a look at the tokens: 2 rows of 100,000 48 -> 29 us)
    const bool all = t1 - t0 > (uint32_t)S;
    if (tid < S / 32) named[tid] = all ? ~0u : 0u;
    if (all)
        for (int i = tid; i < S; i += W) count[i] = which[i] = 0;
    __syncthreads();
    if (!all) {
        const auto name = [&](uint32_t, int id) {
            atomicOr(&named[id / 32], 1u << (id % 32));
            count[id] = which[id] = 0;
        };
        each(a.r.tokens, t0, t1, name);
        each(a.r.bias_ids, b0, b1, name);
        __syncthreads();
    }
    const uint32_t prompt = a.r.n_prompt ? a.r.n_prompt[row] : 0;
    each(a.r.tokens, t0, t1, [&](uint32_t i, int id) {
        if (i - t0 >= prompt) atomicAdd(&count[id], 1u);
        else if (!(count[id] >> 31)) atomicOr(&count[id], 0x80000000u);
    });
    each(a.r.bias_ids, b0, b1, [&](uint32_t i, int id) { atomicMax(&which[id], i - b0 + 1); });
    __syncthreads();
    if (at >= a.vocab) return;
    const int64_t grammar = !a.r.mask ? -1 : a.r.mask_of ? (int64_t)a.r.mask_of[row] : (int64_t)row;
    uint32_t allowed = 0xffu;
    if (grammar >= 0) allowed = grammar < (int64_t)a.r.mask_rows ? a.r.mask[(size_t)grammar * a.r.mask_ld + at / 32] >> (at % 32) : 0u;
    const int c0 = N * tid;
    const uint32_t changed = (named[c0 / 32] >> (c0 % 32)) & 0xffu;
    if (changed) {
        const float rep = a.r.repetition ? a.r.repetition[row] : 1.0f;
        const float presence = a.r.presence ? a.r.presence[row] : 0.0f, frequency = a.r.frequency ? a.r.frequency[row] : 0.0f;
#pragma unroll
        for (int i = 0; i < N; i++) {
            if (!(changed >> i & 1)) continue;
            float y = (float)v[i];
            const uint32_t n = count[c0 + i], w = which[c0 + i], times = n & 0x7fffffffu;
            if (n) y = y > 0.0f ? y / rep : y * rep;
            if (times) y = y - frequency * (float)times - presence;
            if (w) y += a.r.bias[b0 + w - 1];
            v[i] = (T)y;
        }
    }
#pragma unroll
    for (int i = 0; i < N; i++)
        if (!(allowed >> i & 1)) v[i] = (T)-INFINITY;
    if (at + N <= a.vocab) __builtin_nontemporal_store(v, reinterpret_cast<Chunk*>(out + at));
    else
#pragma unroll
        for (int i = 0; i < N; i++)
            if (at + i < a.vocab) out[at + i] = v[i];
}

}  // namespace yl

using namespace yl;

extern "C" yl_status yl_adjust_logits(void* out, size_t out_ld, const void* logits, size_t ld, int32_t dtype, size_t rows, size_t vocab,
                                      const yl_logit_rules* rules, void* stream) {
    const auto refuse = [](const char* what, yl_status st = YL_ERR_ARG) { set_error(what); return st; };
    if (dtype != YL_T_F32 && dtype != YL_T_F16 && dtype != YL_T_BF16) return refuse("adjust_logits: logits are f32, f16 or bf16", YL_ERR_FORMAT);
    if (!rules) return refuse("adjust_logits: no rules");
    if (!vocab || vocab >= (1ull << 31) || ld < vocab || out_ld < vocab) return refuse("adjust_logits: a vocabulary from 1 to below 2^31, rows at least as far apart");
    if (rows >= (1ull << 31)) return refuse("adjust_logits: fewer than 2^31 rows", YL_ERR_RANGE);
    const yl_logit_rules& r = *rules;
    if (!r.tokens != !r.token_start && r.n_tokens) return refuse("adjust_logits: tokens and token_start, or neither");
    if (r.n_tokens && !r.tokens) return refuse("adjust_logits: n_tokens without tokens");
    if (r.n_tokens >= (1u << 31) || r.n_biases >= (1u << 31)) return refuse("adjust_logits: fewer than 2^31 tokens and biases", YL_ERR_RANGE);
    if (r.n_biases && (!r.bias_ids || !r.bias || !r.bias_start)) return refuse("adjust_logits: bias_ids, bias and bias_start, or no biases");
    if (r.mask && (r.mask_ld < (vocab + 31) / 32 || (!r.mask_of && r.mask_rows < rows)))
        return refuse("adjust_logits: masks of a bit per id, and one per row or mask_of");
    if (rows == 0) return YL_OK;
    if (!logits || !out || ((uintptr_t)logits | (uintptr_t)out) % (dtype == YL_T_F32 ? 4 : 2)) return refuse("adjust_logits: no logits or no out, or not aligned to their type");
    if (logits == out && ld != out_ld) return refuse("adjust_logits: in place, ld and out_ld are the same");
    RuleArgs a{logits, out, vocab, ld, out_ld, 0, r};
    if (!r.n_tokens) a.r.token_start = nullptr;
    if (!r.n_biases) a.r.bias_start = nullptr;
    auto k = dtype == YL_T_F32 ? k_logit_rules<float> : dtype == YL_T_F16 ? k_logit_rules<_Float16> : k_logit_rules<__bf16>;
    for (; a.row0 < rows; a.row0 += 65535) {
        hipLaunchKernelGGL(k, dim3((unsigned)((vocab + kRuleStretch - 1) / kRuleStretch), (unsigned)std::min<size_t>(rows - a.row0, 65535)), dim3(kRuleThreads), 0,
                           (hipStream_t)stream, a);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) {
            set_error(std::string("adjust_logits launch: ") + hipGetErrorString(e));
            return YL_ERR_HIP;
        }
    }
    return YL_OK;
}
