// Log probabilities of given tokens, with the entropy of each row's distribution and its most probable tokens.
//
// For a row x of logits: log p_i = x_i - m - ln Z with m the largest logit and Z = sum e^(x_i - m); entropy = ln Z - sum e^(x_i - m) (x_i - m) / Z.
// Tokens of probability zero (a logit of minus infinity) add nothing. A row in which nothing has a probability (all minus infinity), or
// that holds a NaN or plus infinity, has NaN for all of them. The most probable tokens come in falling order, of equal logits the lower id
// first (0 and -0 are equal; a NaN comes last of all).
#include "common.cuh"

constexpr int LP_THREADS = 512;
constexpr int LP_MAX_TOP = 32;

// A logit as a whole number of the same order; ties between ids are broken by the low half of (order, ~id).
__device__ __forceinline__ unsigned lp_order(float x) {
    const unsigned b = __float_as_uint(x);
    if ((b & 0x7fffffffu) > 0x7f800000u) return 0u;                     // NaN
    if ((b & 0x7fffffffu) == 0u) return 0x80000000u;                    // 0 and -0
    return b >> 31 ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ unsigned long long lp_key(float x, int id) { return (unsigned long long)lp_order(x) << 32 | (unsigned)~id; }

__device__ __forceinline__ float lp_block_sum(float v, float* s) {
    v = gb_warp_sum(v);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
    __syncthreads();
    float sum = 0.f;
    for (int w = 0; w < LP_THREADS / 32; ++w) sum += s[w];
    return sum;
}

template <typename T>
__global__ void __launch_bounds__(LP_THREADS) logprobs_kernel(const T* __restrict__ logits, long long stride, const int* __restrict__ tokens,
                                                              float* __restrict__ logprob, float* __restrict__ entropy,
                                                              float* __restrict__ top_logprob, int* __restrict__ top_ids, int top, int vocab) {
    __shared__ float s[LP_THREADS / 32];
    __shared__ unsigned long long sk[LP_THREADS / 32];
    gb_pdl_launch_dependents();
    gb_pdl_wait();
    const int row = blockIdx.x;
    const T* x = logits + (size_t)row * stride;
    float m = -INFINITY;
    for (int i = threadIdx.x; i < vocab; i += LP_THREADS) m = fmaxf(m, gb_to_float(x[i]));
    m = gb_warp_max(m);
    if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = m;
    __syncthreads();
    for (int w = 0; w < LP_THREADS / 32; ++w) m = fmaxf(m, s[w]);
    float z = 0.f, h = 0.f;
    for (int i = threadIdx.x; i < vocab; i += LP_THREADS) {
        const float d = gb_to_float(x[i]) - m, e = expf(d);
        z += e;
        if (e > 0.f) h = fmaf(e, d, h);
    }
    z = lp_block_sum(z, s);
    h = lp_block_sum(h, s);
    const float norm = logf(z);
    if (threadIdx.x == 0) {
        const int token = tokens[row];
        logprob[row] = token >= 0 && token < vocab ? gb_to_float(x[token]) - m - norm : __uint_as_float(0x7fc00000u);
        if (entropy) entropy[row] = norm - h / z;
    }
    unsigned long long last = ~0ull;
    for (int k = 0; k < top; ++k) {
        unsigned long long best = 0;
        for (int i = threadIdx.x; i < vocab; i += LP_THREADS) {
            const unsigned long long key = lp_key(gb_to_float(x[i]), i);
            if (key < last && key > best) best = key;
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            const unsigned long long other = __shfl_xor_sync(0xffffffffu, best, o);
            if (other > best) best = other;
        }
        __syncthreads();
        if ((threadIdx.x & 31) == 0) sk[threadIdx.x >> 5] = best;
        __syncthreads();
        for (int w = 0; w < LP_THREADS / 32; ++w)
            if (sk[w] > best) best = sk[w];
        last = best;
        if (threadIdx.x == 0) {
            const int id = (int)~(unsigned)best;
            top_ids[(size_t)row * top + k] = id;
            if (top_logprob) top_logprob[(size_t)row * top + k] = gb_to_float(x[id]) - m - norm;
        }
    }
}

GB_EXPORT int gb_token_logprobs(const void* logits, int dtype, long long stride, const int* tokens, float* logprob, float* entropy,
                                float* top_logprob, int* top_ids, int top, int rows, int vocab, cudaStream_t stream) {
    GB_REQUIRE(rows >= 0 && vocab > 0 && (rows <= 1 || stride >= vocab), "gb_token_logprobs: bad sizes rows=%d vocab=%d", rows, vocab);
    GB_REQUIRE(top >= 0 && top <= LP_MAX_TOP && top <= vocab, "gb_token_logprobs: %d alternatives of %d tokens (at most %d)", top, vocab, LP_MAX_TOP);
    GB_REQUIRE(dtype == GB_F32 || dtype == GB_BF16, "gb_token_logprobs: unsupported dtype %d", dtype);
    if (rows == 0) return 0;
    GB_REQUIRE(logits && tokens && logprob && (top == 0 || top_ids), "gb_token_logprobs: a tensor is missing");
    const dim3 grid(rows), block(LP_THREADS);
    if (dtype == GB_F32)
        gb_launch(GB_PDL_ELEMENTWISE, logprobs_kernel<float>, grid, block, 0, stream, (const float*)logits, stride, tokens, logprob, entropy,
                  top_logprob, top_ids, top, vocab);
    else
        gb_launch(GB_PDL_ELEMENTWISE, logprobs_kernel<__nv_bfloat16>, grid, block, 0, stream, (const __nv_bfloat16*)logits, stride, tokens, logprob,
                  entropy, top_logprob, top_ids, top, vocab);
    return gb_check_launch("gb_token_logprobs");
}
