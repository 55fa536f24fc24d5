// Log probabilities of given tokens, with the entropy of each row's distribution and its most probable tokens.
//
// For a row x of logits and any reference r: with Z = sum e^(x_i - r) and H = sum e^(x_i - r) (x_i - r), log p_i = x_i - r - ln Z and the
// entropy is ln Z - H / Z; when the reference rises by a, Z becomes Z e^-a and H becomes (H - a Z) e^-a. Tokens of probability zero (a logit of
// minus infinity) add nothing. A row in which nothing has a probability (all minus infinity), or that holds a NaN or plus infinity, has NaN
// for all of them. The most probable tokens come in falling order, of equal logits the lower id first (0 and -0 are equal; NaN comes last).
//
// What bounds it is reading the logits, once. A block takes a row (or, of few rows, a share of one: the blocks of a cluster add up) in
// tiles of 4,096; the next tile's loads are under way while a tile is worked on. Every thread keeps a reference, Z and H of its own. The
// most probable tokens are found in the same pass: k numbers at least as large as a threshold are known to exist if it is the k-th
// largest of the threads' maxima (four of each warp are looked at); only what reaches it is written down (some k numbers in the first tile,
// fewer and fewer as the threshold rises, which it does in tiles 0, 3, 15 ...), and one warp picks the k largest of that. Behind the tile that set it a number
// has to be larger, since equal ones of higher ids come too late. A row that leaves more than 2,048 candidates (one that only rises, or that holds thousands of
// equal largest numbers) is searched k times instead.
// Measured: 2,048 rows of 49,152 float32 (403 MB) with 20 alternatives 89 us, 4.5 TB/s; 1,000 rows of 100,003 bfloat16 that start at odd places, with 5, 62 us.
// No unit is full (20 alternatives: issue slots 63 %, exponentials 35 %, memory 47 %): warps wait at the barriers of the thresholds and of the choice, and
// for loads; without alternatives 67 us are 6.0 TB/s.
#include "common.cuh"

#include <cooperative_groups.h>

// (2,048 rows of 49,152 float32 with 20 alternatives, threads a block and blocks a multiprocessor: 256 and 3 / 4 / 5 105 / 89 / 92 us, 512 and 2
// 112; thresholds in tiles 0, 1, 3, 7 ... 90, in the first alone 108; without alternatives 67)
constexpr int LP_THREADS = 256, LP_WARPS = LP_THREADS / 32;
constexpr int LP_MAX_TOP = 32;
constexpr int LP_EACH = 16;             // numbers of a thread and tile
constexpr int LP_KEEP = 2048;            // candidates

// A logit as a whole number of the same order; ties between ids are broken by the low half of (order, ~id).
__device__ __forceinline__ unsigned lp_order(float x) {
    const unsigned b = __float_as_uint(x);
    if ((b & 0x7fffffffu) > 0x7f800000u) return 0u;                     // NaN
    if ((b & 0x7fffffffu) == 0u) return 0x80000000u;                    // 0 and -0
    return b >> 31 ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ unsigned long long lp_key(float x, int id) { return (unsigned long long)lp_order(x) << 32 | (unsigned)~id; }
__device__ __forceinline__ float lp_number(unsigned order) {            // the logit again (-0 as 0)
    return order == 0u ? __uint_as_float(0x7fc00000u) : order >> 31 ? __uint_as_float(order & 0x7fffffffu) : __uint_as_float(~order);
}
__device__ __forceinline__ float lp_max_nan(float a, float b) {         // NaN where a is one
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float lp_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// The next smaller float32 of a number.
__device__ __forceinline__ float lp_below(float x) {
    const int b = __float_as_int(x);
    return x == 0.f ? __uint_as_float(0x80000001u) : __int_as_float(b < 0 ? b + 1 : b - 1);
}

// The largest key of a warp's.
__device__ __forceinline__ unsigned long long lp_warp_max(unsigned long long key) {
    const unsigned high = __reduce_max_sync(0xffffffffu, (unsigned)(key >> 32));
    const unsigned low = __reduce_max_sync(0xffffffffu, (unsigned)(key >> 32) == high ? (unsigned)key : 0u);
    return (unsigned long long)high << 32 | low;
}

template <typename T> struct LpVec;        // 16 bytes of logits
template <> struct LpVec<float> {
    static constexpr int N = 4;
    static __device__ __forceinline__ void unpack(const uint4& v, float (&x)[4]) {
        x[0] = __uint_as_float(v.x); x[1] = __uint_as_float(v.y); x[2] = __uint_as_float(v.z); x[3] = __uint_as_float(v.w);
    }
    static __device__ __forceinline__ uint4 nothing() { return make_uint4(0xff800000u, 0xff800000u, 0xff800000u, 0xff800000u); }
};
template <> struct LpVec<__nv_bfloat16> {
    static constexpr int N = 8;
    static __device__ __forceinline__ void unpack(const uint4& v, float (&x)[8]) {
        const unsigned w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[2 * i] = __uint_as_float(w[i] << 16);
            x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
    }
    static __device__ __forceinline__ uint4 nothing() { return make_uint4(0xff80ff80u, 0xff80ff80u, 0xff80ff80u, 0xff80ff80u); }
};

struct LpArgs {
    const void* logits;
    long long stride;
    const int* tokens;
    float* logprob;
    float* entropy;
    float* top_logprob;
    int* top_ids;
    int top, vocab, shares;
};

struct LpShared {
    float r[LP_WARPS], z[LP_WARPS], h[LP_WARPS];
    unsigned maxima[LP_MAX_TOP];
    float level;
    float all[3];                              // of the block: reference, Z, H
    int count, found;
    unsigned long long best[LP_MAX_TOP];        // of the block, falling
    unsigned long long keep[LP_KEEP];
};

// The running sums of a thread. r: the reference, minus infinity while all logits were.
struct LpSums {
    float r = -INFINITY, z = 0.f, h = 0.f;
    __device__ __forceinline__ void rise(float to) {
        if (to > r) {
            const float d = r == -INFINITY ? 0.f : r - to, f = lp_exp2(d * 1.4426950408889634f);
            h = f * fmaf(d, z, h);
            z *= f;
            r = to;
        }
    }
    // (a token that is e^-150 times as likely as the likeliest adds nothing to a float32 sum of them)
    __device__ __forceinline__ void add(float x, float from) {
        const float d = lp_max_nan(x - from, -150.f), e = lp_exp2(d * 1.4426950408889634f);
        z += e;
        h = fmaf(e, d, h);
    }
    __device__ __forceinline__ void join(float ro, float zo, float ho) {
        if (ro == -INFINITY) { z += zo; h += ho; return; }          // (nothing, or NaN)
        rise(ro);
        const float d = ro - r, f = lp_exp2(d * 1.4426950408889634f);
        z = fmaf(zo, f, z);
        h = fmaf(f, fmaf(d, zo, ho), h);
    }
};

// How large a number has to be so that `top` are at least as large: the top-th largest of each warp's four largest threads' maxima.
__device__ __forceinline__ float lp_level(LpShared& s, float most, int top) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    unsigned left = lp_order(most);
#pragma unroll
    for (int i = 0; i < LP_MAX_TOP / LP_WARPS; ++i) {
        const unsigned level = __reduce_max_sync(0xffffffffu, left);
        const unsigned who = __ballot_sync(0xffffffffu, left == level);
        if (lane == __ffs(who) - 1) left = 0;
        if (lane == 0) s.maxima[warp * (LP_MAX_TOP / LP_WARPS) + i] = level;
    }
    __syncthreads();
    if (warp == 0) {
        const unsigned mine = s.maxima[lane];
        int before = 0;                         // how many come before this one in falling order
#pragma unroll
        for (int i = 0; i < LP_MAX_TOP; ++i) {
            const unsigned other = __shfl_sync(0xffffffffu, mine, i);
            before += other > mine || (other == mine && i < lane);
        }
        if (before == top - 1) s.level = lp_number(mine);
    }
    __syncthreads();
    return s.level;
}

template <typename T>
__global__ void __launch_bounds__(LP_THREADS, 4) logprobs_kernel(const LpArgs a) {
    using Vec = LpVec<T>;
    constexpr int N = Vec::N, LP_FLY = LP_EACH / N, TILE = LP_THREADS * LP_FLY;         // (of 16-byte pieces)
    constexpr int AHEAD = 16 / sizeof(T) / 4;                                            // tiles that are under way beside the one worked on
    __shared__ LpShared s;
    namespace cg = cooperative_groups;
    const int shares = a.shares, share = blockIdx.x % shares, row = blockIdx.x / shares, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    gb_pdl_launch_dependents();
    gb_pdl_wait();
    const T* x = (const T*)a.logits + (size_t)row * a.stride;
    const int token = tid == 0 && share == 0 ? a.tokens[row] : -1;
    const float own = token >= 0 && token < a.vocab ? gb_to_float(x[token]) : 0.f;
    if (tid == 0) { s.count = 0; s.found = 0; }
    __syncthreads();

    // The row's 16-byte pieces, in equal shares; what lies before the first of them goes to the first share, behind the last one to the last.
    const int lead = min(a.vocab, (int)((16 - ((uintptr_t)x & 15)) & 15) / (int)sizeof(T));
    const int pieces = (a.vocab - lead) / N, begin = (int)((long long)pieces * share / shares), end = (int)((long long)pieces * (share + 1) / shares);
    const uint4* body = reinterpret_cast<const uint4*>(x + lead);
    const int lo = share == 0 ? 0 : lead + begin * N, hi = share == shares - 1 ? a.vocab : lead + end * N;      // ids of this block
    LpSums sums;
    float most = -INFINITY, level = -INFINITY;
    auto keep = [&](float v, int id) {
        const int at = atomicAdd(&s.count, 1);
        if (at < LP_KEEP) s.keep[at] = lp_key(v, id);
    };
    uint4 raw[AHEAD][LP_FLY];
    auto load = [&](int tile, uint4 (&to)[LP_FLY]) {
#pragma unroll
        for (int u = 0; u < LP_FLY; ++u) {
            const int i = begin + tile * TILE + u * LP_THREADS + tid;
            to[u] = i < end ? __ldcs(body + i) : Vec::nothing();
        }
    };
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) load(i, raw[i]);
    // the ragged ends, up to N - 1 numbers each, one a thread
    const int head = share == 0 ? lead : 0, tail = share == shares - 1 ? a.vocab - lead - pieces * N : 0;
    float odd = -INFINITY;
    int odd_id = -1;
    if (tid < head + tail) {
        odd_id = tid < head ? tid : lead + pieces * N + tid - head;
        odd = gb_to_float(x[odd_id]);
        sums.rise(odd);
        sums.add(odd, sums.r == -INFINITY ? 0.f : sums.r);
        if (tid < head) most = odd;             // (what has the highest ids says nothing about equal numbers before it)
    }
    const int tiles = max(1, (end - begin + TILE - 1) / TILE);
    for (int tile = 0; tile < tiles; ++tile) {
        float v[LP_FLY][N], ups[LP_FLY], up = -INFINITY;
#pragma unroll
        for (int u = 0; u < LP_FLY; ++u) {
            Vec::unpack(raw[0][u], v[u]);
            ups[u] = v[u][0];
#pragma unroll
            for (int e = 1; e < N; ++e) ups[u] = fmaxf(ups[u], v[u][e]);
            up = fmaxf(up, ups[u]);
        }
#pragma unroll
        for (int i = 0; i + 1 < AHEAD; ++i)
#pragma unroll
            for (int u = 0; u < LP_FLY; ++u) raw[i][u] = raw[i + 1][u];
        load(tile + AHEAD, raw[AHEAD - 1]);
        sums.rise(up);
        const float from = sums.r == -INFINITY ? 0.f : sums.r;
#pragma unroll
        for (int u = 0; u < LP_FLY; ++u)
#pragma unroll
            for (int e = 0; e < N; ++e) sums.add(v[u][e], from);
        if (a.top) {
            most = fmaxf(most, up);
            const bool fresh = (tile & (tile + 1)) == 0 && ((tile + 1) & 0x55555555) != 0;      // 0, 3, 15 ...
            if (fresh) {
                level = lp_level(s, most, a.top);
                if (tile == 0 && odd_id >= 0 && odd >= level && odd > -INFINITY) keep(odd, odd_id);
            }
            // (at the tile that set it a number at the threshold counts; minus infinity never does)
            const float above = fresh && level > -INFINITY ? lp_below(level) : level;
            if (up > above) {
#pragma unroll
                for (int u = 0; u < LP_FLY; ++u)
                    if (ups[u] > above)
#pragma unroll
                        for (int e = 0; e < N; ++e)
                            if (v[u][e] > above) keep(v[u][e], lead + (begin + tile * TILE + u * LP_THREADS + tid) * N + e);
            }
        }
    }
    // ---- the block's sums
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const float r = __shfl_xor_sync(0xffffffffu, sums.r, o), z = __shfl_xor_sync(0xffffffffu, sums.z, o), h = __shfl_xor_sync(0xffffffffu, sums.h, o);
        sums.join(r, z, h);
    }
    if (lane == 0) { s.r[warp] = sums.r; s.z[warp] = sums.z; s.h[warp] = sums.h; }
    __syncthreads();
    const bool searched = a.top && s.count > LP_KEEP;
    if (searched) {                             // k times through the block's share of the row
        unsigned long long last = ~0ull;
        for (int k = 0; k < a.top; ++k) {
            unsigned long long best = 0;
            for (int i = lo + tid; i < hi; i += LP_THREADS) {
                const float v = gb_to_float(x[i]);
                const unsigned long long key = lp_key(v, i);
                if (v > -INFINITY && key < last && key > best) best = key;
            }
            best = lp_warp_max(best);
            __syncthreads();
            if (lane == 0) s.keep[warp] = best;
            __syncthreads();
#pragma unroll
            for (int w = 0; w < LP_WARPS; ++w)
                if (s.keep[w] > best) best = s.keep[w];
            if (best == 0) break;
            last = best;
            if (tid == 0) { s.best[k] = best; s.found = k + 1; }
        }
        __syncthreads();
    }
    if (warp == 0) {
        LpSums all;
        if (lane < LP_WARPS) { all.r = s.r[lane]; all.z = s.z[lane]; all.h = s.h[lane]; }
#pragma unroll
        for (int o = LP_WARPS / 2; o > 0; o >>= 1) {
            const float r = __shfl_xor_sync(0xffffffffu, all.r, o), z = __shfl_xor_sync(0xffffffffu, all.z, o), h = __shfl_xor_sync(0xffffffffu, all.h, o);
            all.join(r, z, h);
        }
        if (lane == 0) { s.all[0] = all.r; s.all[1] = all.z; s.all[2] = all.h; }
        if (a.top && !searched) {
            const int count = s.count;
            constexpr int HELD = 4;             // a lane's candidates that stay in registers: mostly all of them
            unsigned long long held[HELD], last = ~0ull;
#pragma unroll
            for (int i = 0; i < HELD; ++i) held[i] = lane + 32 * i < count ? s.keep[lane + 32 * i] : 0;
            for (int k = 0; k < a.top; ++k) {
                unsigned long long best = 0;
#pragma unroll
                for (int i = 0; i < HELD; ++i)
                    if (held[i] < last && held[i] > best) best = held[i];
                for (int i = lane + 32 * HELD; i < count; i += 32) {
                    const unsigned long long key = s.keep[i];
                    if (key < last && key > best) best = key;
                }
                best = lp_warp_max(best);
                if (best == 0) break;
                last = best;
                if (lane == 0) { s.best[k] = best; s.found = k + 1; }
            }
        }
    }
    // ---- the row's: the first block of a cluster takes what the others have
    if (shares > 1) cg::this_cluster().sync();
    if (share == 0 && warp == 0) {
        __syncwarp();
        LpSums all;
        auto of = [&](int b) -> const LpShared* { return shares > 1 ? cg::this_cluster().map_shared_rank(&s, b) : &s; };
        if (lane < shares) { const LpShared* o = of(lane); all.r = o->all[0]; all.z = o->all[1]; all.h = o->all[2]; }
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) {
            const float r = __shfl_xor_sync(0xffffffffu, all.r, o), z = __shfl_xor_sync(0xffffffffu, all.z, o), h = __shfl_xor_sync(0xffffffffu, all.h, o);
            all.join(r, z, h);
        }
        const float nan = __uint_as_float(0x7fc00000u);
        const bool none = !(all.r > -INFINITY) || all.r == INFINITY;
        const float r = __shfl_sync(0xffffffffu, none ? nan : all.r, 0), norm = __shfl_sync(0xffffffffu, logf(all.z), 0);
        if (lane == 0) {
            a.logprob[row] = token >= 0 && token < a.vocab ? own - r - norm : nan;
            if (a.entropy) a.entropy[row] = none ? nan : norm - all.h / all.z;
        }
        if (a.top) {
            // lane b walks down block b's list; the k-th largest goes to lane k
            unsigned long long out = 0;
            int k = 0;
            if (shares == 1) {
                k = s.found;
                if (lane < k) out = s.best[lane];
            } else {
                const LpShared* mine = of(lane < shares ? lane : 0);
                const int has = lane < shares ? mine->found : 0;
                int next = 0;
                unsigned long long key = has > 0 ? mine->best[0] : 0;
                for (; k < a.top; ++k) {
                    const unsigned long long best = lp_warp_max(key);
                    if (best == 0) break;
                    if (lane == k) out = best;
                    if (key == best) key = ++next < has ? mine->best[next] : 0;
                }
            }
            // fewer tokens have a probability: the first ones that have none, then those that are NaN
            for (int pass = 0; pass < 2 && k < a.top; ++pass)
                for (int i0 = 0; i0 < a.vocab && k < a.top; i0 += 32) {
                    const int i = i0 + lane;
                    const float v = i < a.vocab ? gb_to_float(x[i]) : 0.f;
                    unsigned hits = __ballot_sync(0xffffffffu, i < a.vocab && (pass == 0 ? v == -INFINITY : v != v));
                    for (; hits && k < a.top; hits &= hits - 1, ++k)
                        if (lane == k) out = lp_key(pass == 0 ? -INFINITY : nan, i0 + __ffs(hits) - 1);
                }
            if (lane < a.top) {
                a.top_ids[(size_t)row * a.top + lane] = (int)~(unsigned)out;
                if (a.top_logprob) a.top_logprob[(size_t)row * a.top + lane] = lp_number((unsigned)(out >> 32)) - r - norm;
            }
        }
    }
    if (shares > 1) cg::this_cluster().sync();   // (its memory is read until here)
}

// top_ids [rows, top] (top 0: none), top_logprob and entropy may be missing. Rows `stride` numbers apart.
GB_EXPORT int gb_token_logprobs(const void* logits, int dtype, long long stride, const int* tokens, float* logprob, float* entropy,
                                float* top_logprob, int* top_ids, int top, int rows, int vocab, cudaStream_t stream) {
    GB_REQUIRE(rows >= 0 && vocab > 0 && (rows <= 1 || stride >= vocab), "gb_token_logprobs: bad sizes rows=%d vocab=%d", rows, vocab);
    GB_REQUIRE(top >= 0 && top <= LP_MAX_TOP && top <= vocab, "gb_token_logprobs: %d alternatives of %d tokens (at most %d)", top, vocab, LP_MAX_TOP);
    GB_REQUIRE(dtype == GB_F32 || dtype == GB_BF16, "gb_token_logprobs: unsupported dtype %d", dtype);
    GB_REQUIRE(rows < (1 << 28), "gb_token_logprobs: %d rows are too many for one launch", rows);
    if (rows == 0) return 0;
    GB_REQUIRE(logits && tokens && logprob && (top == 0 || top_ids), "gb_token_logprobs: a tensor is missing");
    LpArgs a = {logits, stride, tokens, logprob, entropy, top_logprob, top_ids, top, vocab, 1};
    const int size = dtype == GB_F32 ? 4 : 2;
    // Shares of at least 16 KB of a row while all fit at once, two a multiprocessor: rows of 128,256 float32 in 1 / 2 / 4 / 8 shares, one row 20.4 /
    // 15.9 / 12.5 / 10.3 us, 37 rows 28.9 / 19.9 / 17.0 / 14.5, 148 rows 30.6 / 23.5 / 31.3 / 36.3; rows of 8,192, one 6.7 / 6.3 / 6.3 / 6.4, 148 rows
    // 7.2 / 7.3 / 13.6 / 20.7.
    int shares = 8;
    while (shares > 1 && ((long long)rows * shares > 2 * 148 || (long long)vocab * size < shares * 16384ll)) shares /= 2;
    cudaLaunchConfig_t cfg = {};
    a.shares = shares;
    cfg.gridDim = dim3(shares * rows);
    cfg.blockDim = dim3(LP_THREADS);
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    int na = 0;
    if (gb_pdl_enabled() & GB_PDL_ELEMENTWISE) {
        attr[na].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[na].val.programmaticStreamSerializationAllowed = 1;
        ++na;
    }
    if (shares > 1) {
        attr[na].id = cudaLaunchAttributeClusterDimension;
        attr[na].val.clusterDim.x = shares;
        attr[na].val.clusterDim.y = attr[na].val.clusterDim.z = 1;
        ++na;
    }
    cfg.attrs = attr;
    cfg.numAttrs = na;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, dtype == GB_F32 ? logprobs_kernel<float> : logprobs_kernel<__nv_bfloat16>, a);
    if (e != cudaSuccess) {
        gb_set_error("gb_token_logprobs: launch failed: %s", cudaGetErrorString(e));
        return 2;
    }
    return gb_check_launch("gb_token_logprobs");
}
