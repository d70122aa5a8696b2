// yl_logprobs.hip -- log probabilities of given tokens, the entropy and the
// most probable alternatives of rows of logits.  No counterpart in the
// reference (sampler.rs holds one row of probabilities on the host).
#include <hip/hip_runtime.h>

#include <math.h>

#include "../../include/yallma3.h"
#include "yl_device.h"
#include "yl_internal.h"

namespace yl {

constexpr int kTopMost = 32;

// A value's place in the order of the top list: NaN last, -0 with +0.
__device__ __forceinline__ uint32_t order_key(float x) {
    if (x != x) return 0u;
    const uint32_t b = __float_as_uint(x == 0.0f ? 0.0f : x);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

// One workgroup per row: the maximum, the sums, then one pass per top entry.
template <typename T>
__global__ __launch_bounds__(256) void k_token_logprobs(const T* x, size_t vocab, size_t ld, const uint32_t* tokens,
                                                        float* logprob, float* entropy, int top, uint32_t* top_ids,
                                                        float* top_logprobs) {
    __shared__ float rf[4], rg[4];
    __shared__ unsigned long long rk[4];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const size_t r = blockIdx.x;
    const T* row = x + r * ld;
    const auto key = [&](size_t i) { return ((unsigned long long)order_key((float)row[i]) << 32) | (uint32_t)~(uint32_t)i; };
    float m = -INFINITY;
    unsigned long long kmax = 0;
    for (size_t i = tid; i < vocab; i += 256) {
        m = fmaxf(m, (float)row[i]);
        const unsigned long long k = key(i);
        if (k > kmax) kmax = k;
    }
    for (int off = 32; off > 0; off >>= 1) {
        m = fmaxf(m, __shfl_xor(m, off, 64));
        const unsigned long long o = __shfl_xor(kmax, off, 64);
        if (o > kmax) kmax = o;
    }
    if (lane == 0) { rf[wave] = m; rk[wave] = kmax; }
    __syncthreads();
    m = fmaxf(fmaxf(rf[0], rf[1]), fmaxf(rf[2], rf[3]));
    for (int w = 0; w < 4; w++)
        if (rk[w] > kmax) kmax = rk[w];
    __syncthreads();
    // the sums over all but one holder of the maximum, whose weight is 1
    const uint32_t first = ~(uint32_t)kmax;
    float z = 0.0f, t = 0.0f;
    for (size_t i = tid; i < vocab; i += 256) {
        const float v = (float)row[i];
        const float d = v - m;
        const float e = i == first && d == 0.0f ? 0.0f : v == -INFINITY ? 0.0f : expf(d);
        z += e;
        if (e != 0.0f) t = fmaf(d, e, t);
    }
    for (int off = 32; off > 0; off >>= 1) { z += __shfl_xor(z, off, 64); t += __shfl_xor(t, off, 64); }
    if (lane == 0) { rf[wave] = z; rg[wave] = t; }
    __syncthreads();
    z = (rf[0] + rf[1]) + (rf[2] + rf[3]);
    t = (rg[0] + rg[1]) + (rg[2] + rg[3]);
    const float lz = log1pf(z);
    const bool none = m == -INFINITY && z == 0.0f;
    if (tid == 0) {
        if (logprob) logprob[r] = z != z ? z : tokens[r] >= vocab || none ? -INFINITY : ((float)row[tokens[r]] - m) - lz;
        if (entropy) entropy[r] = none ? 0.0f : lz - t / (1.0f + z);
    }
    unsigned long long last = ~0ull;
    for (int j = 0; j < top; j++) {
        unsigned long long best = 0;
        for (size_t i = tid; i < vocab; i += 256) {
            const unsigned long long k = key(i);
            if (k < last && k > best) best = k;
        }
        for (int off = 32; off > 0; off >>= 1) {
            const unsigned long long o = __shfl_xor(best, off, 64);
            if (o > best) best = o;
        }
        __syncthreads();
        if (lane == 0) rk[wave] = best;
        __syncthreads();
        for (int w = 0; w < 4; w++)
            if (rk[w] > best) best = rk[w];
        last = best;
        if (tid == 0) {
            const uint32_t id = ~(uint32_t)best;
            top_ids[r * top + j] = id;
            top_logprobs[r * top + j] = none ? -INFINITY : ((float)row[id] - m) - lz;
        }
    }
}

}  // namespace yl

using namespace yl;

extern "C" {

size_t yl_token_logprobs_workspace(size_t rows, size_t vocab, uint32_t top) {
    return 0;
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
    const size_t need = yl_token_logprobs_workspace(rows, vocab, top);
    if (need && (!workspace || (uintptr_t)workspace % 16)) return refuse("token_logprobs: the workspace has to be there, 16-byte aligned");
    if (workspace_bytes < need) return refuse("token_logprobs: the workspace is smaller than yl_token_logprobs_workspace says", YL_ERR_RANGE);
    const dim3 grid((unsigned)rows), block(256);
    hipStream_t s = (hipStream_t)stream;
    if (dtype == YL_T_F32)
        hipLaunchKernelGGL(k_token_logprobs<float>, grid, block, 0, s, (const float*)logits, vocab, ld, tokens, logprob, entropy, (int)top, top_ids, top_logprobs);
    else if (dtype == YL_T_F16)
        hipLaunchKernelGGL(k_token_logprobs<_Float16>, grid, block, 0, s, (const _Float16*)logits, vocab, ld, tokens, logprob, entropy, (int)top, top_ids, top_logprobs);
    else
        hipLaunchKernelGGL(k_token_logprobs<__bf16>, grid, block, 0, s, (const __bf16*)logits, vocab, ld, tokens, logprob, entropy, (int)top, top_ids, top_logprobs);
    const hipError_t e = hipGetLastError();
    if (e == hipSuccess) return YL_OK;
    set_error(std::string("token_logprobs launch: ") + hipGetErrorString(e));
    return YL_ERR_HIP;
}

}  // extern "C"
