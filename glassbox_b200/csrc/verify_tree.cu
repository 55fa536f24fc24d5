// Verification of a request's tree of drafted tokens against the probabilities that the model gives, from given random numbers.
//
// The walk begins at row 0 of the tree, and at every row it reaches p = softmax(logits / T). Without a drafting model's logits the first token is drawn whose
// sum of probabilities, in the order of the ids, exceeds the row's second random number times the whole (T not above 0: the largest logit, of equal ones the
// lowest id); the walk goes on at the first child that holds this token. With them, q = softmax(draft / T) is what the children were drawn from,
// independently. The leftover after j children that were not taken is r_j = max(r_{j-1} - sum(r_{j-1}) q, 0) = max(p - s_j q, 0) with s_0 = 0,
// s_{j+1} = s_j + sum(r_j): one number holds what was taken away. A child of token x is taken where u sum(r_j) q(x) < r_j(x); behind the last one the token is
// drawn from r as above. So the tokens that come out have the model's distribution, whatever was drafted.
//
// A sum's error would move the border between two tokens, and of 100,000 tokens' borders one lies near most random numbers: weights and sums are held in 64 bits.
// A cluster of blocks walks with a request: each takes a share of the row's segments of 512 tokens, a warp a segment, and keeps their sums; they add up through
// distributed shared memory, and the block whose share holds the target finds the segment and reads it once more. Only rows that the walk reaches are read.
#include "common.cuh"

#include <cooperative_groups.h>

constexpr int VT_THREADS = 256, VT_WARPS = VT_THREADS / 32;
constexpr int VT_SEG = 512, VT_EACH = VT_SEG / 32;      // tokens of a segment, and of a lane
constexpr int VT_MAX_SEGS = 4097;
constexpr int VT_MAX_CLUSTER = 8;

struct VerifyArgs {
    const void* logits;
    long long stride;
    const void* draft;                // or none
    long long draft_stride;
    const int* tokens;
    const int* parents;
    const int* first_row;
    const float* uniform;             // [n, 2]
    const float* temperature;         // [requests]
    int* path;
    int* accepted;
    int* next;
    int n, vocab, blocks;             // blocks of a cluster
};

// What a block tells the others of its share of a row.
struct VtShare {
    double sum;                        // of exp((x - most) / T)
    float most;                        // minus infinity: no token here has a probability
    int wrong;                         // a logit that is NaN or plus infinity
    unsigned long long best;           // the largest logit as (order, ~id)
};

struct VtShared {
    VtShare mine[2][2];                // [turn][p, q]
    double left[2];                    // [turn] of the leftover
    int token[2];                      // [turn] that the block found, -1: none
    double warp_sum[VT_WARPS], warp_sum2[VT_WARPS];
    float warp_most[VT_WARPS], warp_most2[VT_WARPS];
    int warp_wrong[VT_WARPS];
    unsigned long long warp_best[VT_WARPS];
    int child, seen;
};

__device__ __forceinline__ unsigned long long vt_key(float x, int id) {      // NaN is below everything
    const unsigned b = __float_as_uint(x);
    const unsigned order = (b & 0x7fffffffu) > 0x7f800000u ? 0u : (b & 0x7fffffffu) == 0u ? 0x80000000u : b >> 31 ? ~b : b | 0x80000000u;
    return (unsigned long long)order << 32 | (unsigned)~id;
}
__device__ __forceinline__ unsigned long long vt_warp_max(unsigned long long key) {
    const unsigned high = __reduce_max_sync(0xffffffffu, (unsigned)(key >> 32));
    const unsigned low = __reduce_max_sync(0xffffffffu, (unsigned)(key >> 32) == high ? (unsigned)key : 0u);
    return (unsigned long long)high << 32 | low;
}
__device__ __forceinline__ double vt_warp_sum(double v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// A lane's tokens of a segment, 16 bytes at a time: piece u * 32 + lane of the segment's. Segments begin at multiples of 16 bytes: `lead` numbers before the
// row's first one. Tokens outside the row have minus infinity.
template <typename T>
__device__ __forceinline__ void vt_load(const T* x, int lead, int vocab, int seg, float (&v)[VT_EACH]) {
    constexpr int N = 16 / sizeof(T);
    const int lane = threadIdx.x & 31;
    uint4 raw[VT_EACH / N];
    bool whole[VT_EACH / N];
#pragma unroll
    for (int u = 0; u < VT_EACH / N; ++u) {
        const int i = seg * VT_SEG + (u * 32 + lane) * N - lead;
        whole[u] = i >= 0 && i + N <= vocab;
        raw[u] = whole[u] ? *reinterpret_cast<const uint4*>(x + i) : make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int u = 0; u < VT_EACH / N; ++u) {
        const unsigned w[4] = {raw[u].x, raw[u].y, raw[u].z, raw[u].w};
#pragma unroll
        for (int e = 0; e < N; ++e)
            v[u * N + e] = N == 4 ? __uint_as_float(w[e % 4]) : __uint_as_float(e & 1 ? w[(e >> 1) % 4] & 0xffff0000u : w[(e >> 1) % 4] << 16);
        if (!whole[u]) {
#pragma unroll
            for (int e = 0; e < N; ++e) {
                const int i = seg * VT_SEG + (u * 32 + lane) * N + e - lead;
                v[u * N + e] = i >= 0 && i < vocab ? gb_to_float(x[i]) : -INFINITY;
            }
        }
    }
}

template <typename T>
__global__ void __launch_bounds__(VT_THREADS) verify_tree_kernel(const VerifyArgs a) {
    namespace cg = cooperative_groups;
    constexpr int N = 16 / sizeof(T);
    extern __shared__ __align__(16) double vt_mem[];
    __shared__ VtShared sh;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int C = a.blocks, rank = blockIdx.x % C, seq = blockIdx.x / C, vocab = a.vocab;
    const int most_segs = (vocab + N + VT_SEG - 1) / VT_SEG, per = (most_segs + C - 1) / C;
    double* p_sum = vt_mem;                            // of the block's segments: sums of exp((x - most) / T), then (drafted) the leftover's
    double* r_sum = p_sum + per;
    float* p_most = reinterpret_cast<float*>(r_sum + (a.draft ? per : 0));
    gb_pdl_launch_dependents();
    gb_pdl_wait();
    const int row0 = a.first_row[seq], rows = a.first_row[seq + 1] - row0;
    auto cluster_sync = [&]() { if (C > 1) cg::this_cluster().sync(); else __syncthreads(); };
    auto of = [&](int b) -> const VtShared* { return C > 1 ? cg::this_cluster().map_shared_rank(&sh, b) : &sh; };
    if (rows <= 0 || row0 < 0 || row0 > a.n - rows) {  // (the same in all blocks of a cluster)
        if (rank == 0 && tid == 0) { a.accepted[seq] = 0; a.next[seq] = -1; }
        return;
    }
    const float temp = a.temperature[seq];
    const bool draws = temp > 0.f, drafted = draws && a.draft != nullptr;
    const double heat = draws ? 1.0 / (double)temp : 0.0;
    if (rank == 0)
        for (int i = tid; i < rows; i += VT_THREADS) a.path[row0 + i] = i == 0 ? 0 : -1;
    __syncthreads();

    // The block's share of a row: its segments' sums (and largest logits, if `keep`), its own in `to`.
    auto scan = [&](const T* x, bool keep, VtShare& to) {
        const int lead = (int)((uintptr_t)x & 15) / (int)sizeof(T), segs = (lead + vocab + VT_SEG - 1) / VT_SEG;
        const int lo = min(rank * per, segs), hi = min(lo + per, segs);
        float w_most = -INFINITY;
        double w_sum = 0.0;
        bool wrong = false;
        unsigned long long best = 0;
        for (int seg = lo + warp; seg < hi; seg += VT_WARPS) {
            float v[VT_EACH];
            vt_load(x, lead, vocab, seg, v);
            float most = -INFINITY;
#pragma unroll
            for (int i = 0; i < VT_EACH; ++i) {
                most = fmaxf(most, v[i]);
                wrong = wrong || !(v[i] < INFINITY);
                if (!draws) {
                    const int id = seg * VT_SEG + (i / N * 32 + lane) * N + i % N - lead;
                    const unsigned long long key = vt_key(v[i], id);
                    best = key > best && v[i] == v[i] && (unsigned)id < (unsigned)vocab ? key : best;
                }
            }
            if (!draws) continue;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
            double sum = 0.0;
            if (most > -INFINITY && most < INFINITY)
#pragma unroll
                for (int i = 0; i < VT_EACH; ++i) sum += exp(((double)v[i] - (double)most) * heat);
            sum = vt_warp_sum(sum);
            if (keep && lane == 0) { p_sum[seg - lo] = sum; p_most[seg - lo] = most; }
            if (most > w_most) {
                w_sum = w_sum * exp(((double)w_most - (double)most) * heat) + sum;
                w_most = most;
            } else if (most > -INFINITY) {
                w_sum += sum * exp(((double)most - (double)w_most) * heat);
            }
        }
        best = vt_warp_max(best);
        wrong = __any_sync(0xffffffffu, wrong);
        if (lane == 0) { sh.warp_sum[warp] = w_sum; sh.warp_most[warp] = w_most; sh.warp_wrong[warp] = wrong; sh.warp_best[warp] = best; }
        __syncthreads();
        if (tid == 0) {
            float most = -INFINITY;
            double sum = 0.0;
            int bad = 0;
            unsigned long long top = 0;
            for (int w = 0; w < VT_WARPS; ++w) {
                most = fmaxf(most, sh.warp_most[w]);
                bad |= sh.warp_wrong[w];
                top = sh.warp_best[w] > top ? sh.warp_best[w] : top;
            }
            if (most > -INFINITY && most < INFINITY)
                for (int w = 0; w < VT_WARPS; ++w)
                    if (sh.warp_most[w] > -INFINITY) sum += sh.warp_sum[w] * exp(((double)sh.warp_most[w] - (double)most) * heat);
            to.sum = sum; to.most = most; to.wrong = bad; to.best = top;
        }
        __syncthreads();
    };
    // All blocks' shares, behind the cluster's barrier.
    auto whole = [&](int turn, int which, float& most, double& sum) -> bool {
        most = -INFINITY;
        sum = 0.0;
        bool wrong = false;
        for (int b = 0; b < C; ++b) {
            const VtShare* o = &of(b)->mine[turn][which];
            most = fmaxf(most, o->most);
            wrong = wrong || o->wrong;
        }
        if (wrong || !(most > -INFINITY)) return false;
        for (int b = 0; b < C; ++b) {
            const VtShare* o = &of(b)->mine[turn][which];
            if (o->most > -INFINITY) sum += o->sum * exp(((double)o->most - (double)most) * heat);
        }
        return true;
    };
    // The token at which the sum of the weights exceeds `target`: seg_sum(i) is the sum of the block's segment i, weights(seg, w) are a lane's of one. Called by
    // warp 0 of the block in whose share it lies; `before`: the sum of the shares before; `behind`: rounding has left the target behind every weight, the last
    // one is taken.
    auto find = [&](int lo, int hi, int lead, double before, bool behind, double target, auto seg_sum, auto weights) -> int {
        int last = -1;                                 // the last segment that holds a weight
        for (int s0 = lo; s0 < hi; s0 += 32) {
            const double mine = s0 + lane < hi ? seg_sum(s0 + lane - lo) : 0.0;
            double upto = mine;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const double up = __shfl_up_sync(0xffffffffu, upto, o);
                if (lane >= o) upto += up;
            }
            const unsigned some = __ballot_sync(0xffffffffu, mine > 0.0), hit = __ballot_sync(0xffffffffu, mine > 0.0 && !behind && before + upto > target);
            if (hit) {
                const int at = __ffs(hit) - 1;
                before = __shfl_sync(0xffffffffu, before + upto - mine, at);
                last = s0 + at;
                break;
            }
            if (some) last = s0 + 31 - __clz(some);
            before += __shfl_sync(0xffffffffu, upto, 31);
        }
        if (last < 0) return -1;
        double w[VT_EACH];
        weights(last, w);
        int token = -1;
#pragma unroll
        for (int u = 0; u < VT_EACH / N; ++u) {
            double mine = 0.0;
#pragma unroll
            for (int e = 0; e < N; ++e) mine += w[u * N + e];
            double upto = mine;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const double up = __shfl_up_sync(0xffffffffu, upto, o);
                if (lane >= o) upto += up;
            }
            double sum = before + upto - mine;
            int found = -1, held = -1;                 // where the sum passes the target, and the lane's last weight
#pragma unroll
            for (int e = 0; e < N; ++e) {
                const int id = last * VT_SEG + (u * 32 + lane) * N + e - lead;
                sum += w[u * N + e];
                if (w[u * N + e] > 0.0) {
                    held = id;
                    if (found < 0 && sum > target && !behind) found = id;
                }
            }
            const unsigned hit = __ballot_sync(0xffffffffu, found >= 0), some = __ballot_sync(0xffffffffu, held >= 0);
            if (hit) return __shfl_sync(0xffffffffu, found, __ffs(hit) - 1);
            if (some) token = __shfl_sync(0xffffffffu, held, 31 - __clz(some));
            before += __shfl_sync(0xffffffffu, upto, 31);
        }
        return token;
    };

    int cur = 0, kept = 1, token = -1;
    for (int step = 0;; ++step) {                      // (a child lies behind its parent: at most `rows` steps)
        const int turn = step & 1;
        const T* x = (const T*)a.logits + (size_t)(row0 + cur) * a.stride;
        const T* y = drafted ? (const T*)a.draft + (size_t)(row0 + cur) * a.draft_stride : nullptr;
        const int lead = (int)((uintptr_t)x & 15) / (int)sizeof(T), segs = (lead + vocab + VT_SEG - 1) / VT_SEG;
        const int lo = min(rank * per, segs), hi = min(lo + per, segs);
        scan(x, true, sh.mine[turn][0]);
        if (drafted) scan(y, false, sh.mine[turn][1]);
        cluster_sync();
        int child = -1;                                // where the walk goes on
        token = -1;
        // the first row behind `after` that is a child of this one (and holds `like`, if that is a token)
        auto next_child = [&](int after, int like) -> int {
            __syncthreads();
            if (tid == 0) sh.child = rows;
            __syncthreads();
            for (int c = max(cur, after) + 1 + tid; c < rows; c += VT_THREADS)
                if (a.parents[row0 + c] == cur && (like < 0 || a.tokens[row0 + c] == like)) { atomicMin(&sh.child, c); break; }
            __syncthreads();
            return sh.child < rows ? sh.child : -1;
        };
        if (!draws) {
            unsigned long long best = 0;
            for (int b = 0; b < C; ++b) { const unsigned long long o = of(b)->mine[turn][0].best; best = o > best ? o : best; }
            token = best ? (int)~(unsigned)best : -1;
            if (token >= 0) child = next_child(cur, token);
        } else {
            float most, q_most = 0.f;
            double sum, q_sum = 1.0;
            const bool fine = whole(turn, 0, most, sum), q_fine = !drafted || whole(turn, 1, q_most, q_sum);
            const double u = (double)a.uniform[2 * (size_t)(row0 + cur) + 1];
            double away = 0.0, left = 1.0;             // s and sum(r)
            bool drawn_from_left = false;
            if (fine && q_fine && drafted) {
                for (int c = next_child(cur, -1); c >= 0; c = next_child(c, -1)) {
                    const int t = a.tokens[row0 + c];
                    if (t < 0 || t >= vocab) continue;     // (nothing that q could have given)
                    const double p = exp(((double)gb_to_float(x[t]) - (double)most) * heat) / sum, q = exp(((double)gb_to_float(y[t]) - (double)q_most) * heat) / q_sum;
                    const double r = fmax(p - away * q, 0.0);
                    if ((double)a.uniform[2 * (size_t)(row0 + c)] * q * left < r) { child = c; break; }
                    // not taken: what is left without it
                    away += left;
                    drawn_from_left = true;
                    double w_sum = 0.0;
                    for (int seg = lo + warp; seg < hi; seg += VT_WARPS) {
                        float v[VT_EACH];
                        vt_load(x, lead, vocab, seg, v);
                        double s = 0.0;
#pragma unroll
                        for (int i = 0; i < VT_EACH; ++i) {
                            const int id = seg * VT_SEG + (i / N * 32 + lane) * N + i % N - lead;
                            if (v[i] > -INFINITY) s += fmax(exp(((double)v[i] - (double)most) * heat) / sum - away * (exp(((double)gb_to_float(y[id]) - (double)q_most) * heat) / q_sum), 0.0);
                        }
                        s = vt_warp_sum(s);
                        if (lane == 0) r_sum[seg - lo] = s;
                        w_sum += s;
                    }
                    if (lane == 0) sh.warp_sum2[warp] = w_sum;
                    cluster_sync();                    // (the leftover before has been read by all)
                    if (tid == 0) {
                        double s = 0.0;
                        for (int w = 0; w < VT_WARPS; ++w) s += sh.warp_sum2[w];
                        sh.left[0] = s;
                    }
                    cluster_sync();
                    left = 0.0;
                    for (int b = 0; b < C; ++b) left += of(b)->left[0];
                    if (!(left > 0.0)) { drawn_from_left = false; break; }
                }
            }
            if (fine && q_fine && child < 0) {
                // draw: the block whose share holds the target finds the token
                const double target = u * (drawn_from_left ? left : sum);
                double before = 0.0, mine = 0.0;
                int owner = -1, filled = -1;           // (filled: the last block that holds a weight; rounding may leave the target behind it)
                double owner_before = 0.0;
                for (int b = 0; b < C; ++b) {
                    const VtShared* o = of(b);
                    mine = drawn_from_left ? o->left[0] : o->mine[turn][0].most > -INFINITY ? o->mine[turn][0].sum * exp(((double)o->mine[turn][0].most - (double)most) * heat) : 0.0;
                    if (mine > 0.0) {
                        filled = b;
                        if (owner < 0 && before + mine > target) { owner = b; owner_before = before; }
                    }
                    before += mine;
                }
                const bool behind = owner < 0;
                if (behind) owner = filled;
                if (owner == rank && warp == 0) {
                    auto weight = [&](float v) { return v > -INFINITY ? exp(((double)v - (double)most) * heat) : 0.0; };
                    auto p_seg = [&](int i) { return p_most[i] > -INFINITY ? p_sum[i] * exp(((double)p_most[i] - (double)most) * heat) : 0.0; };
                    auto r_seg = [&](int i) { return r_sum[i]; };
                    auto p_weights = [&](int seg, double (&w)[VT_EACH]) {
                        float v[VT_EACH];
                        vt_load(x, lead, vocab, seg, v);
#pragma unroll
                        for (int i = 0; i < VT_EACH; ++i) w[i] = weight(v[i]);
                    };
                    auto r_weights = [&](int seg, double (&w)[VT_EACH]) {
                        float v[VT_EACH];
                        vt_load(x, lead, vocab, seg, v);
#pragma unroll
                        for (int i = 0; i < VT_EACH; ++i) {
                            const int id = seg * VT_SEG + (i / N * 32 + lane) * N + i % N - lead;
                            w[i] = v[i] > -INFINITY ? fmax(weight(v[i]) / sum - away * (exp(((double)gb_to_float(y[id]) - (double)q_most) * heat) / q_sum), 0.0) : 0.0;
                        }
                    };
                    const int found = drawn_from_left ? find(lo, hi, lead, owner_before, behind, target, r_seg, r_weights) : find(lo, hi, lead, owner_before, behind, target, p_seg, p_weights);
                    if (lane == 0) sh.token[turn] = found;
                }
                cluster_sync();
                token = owner >= 0 ? of(owner)->token[turn] : -1;
                if (!drafted && token >= 0) child = next_child(cur, token);
            }
        }
        if (child < 0) break;
        cur = child;
        if (rank == 0 && tid == 0) a.path[row0 + kept] = cur;
        ++kept;
    }
    if (rank == 0 && tid == 0) {
        a.accepted[seq] = kept;
        a.next[seq] = token;
    }
    cluster_sync();                                    // (shared memory is read until here)
}

// logits, draft: [n, vocab] of one type, rows `stride` numbers apart (draft: or none). Everything else as above; path [n], accepted and next [requests].
GB_EXPORT int gb_verify_tree(const void* logits, int dtype, long long stride, const void* draft, long long draft_stride, const int* tokens, const int* parents,
                             const int* first_row, const float* uniform, const float* temperature, int* path, int* accepted, int* next, int n, int num_seqs,
                             int vocab, cudaStream_t stream) {
    GB_REQUIRE(n >= 0 && num_seqs >= 0 && vocab > 0 && (n <= 1 || stride >= vocab) && (draft == nullptr || n <= 1 || draft_stride >= vocab), "gb_verify_tree: bad sizes n=%d vocab=%d", n, vocab);
    GB_REQUIRE(vocab <= (VT_MAX_SEGS - 1) * VT_SEG, "gb_verify_tree: a vocabulary of %d is not built (%d)", vocab, (VT_MAX_SEGS - 1) * VT_SEG);
    GB_REQUIRE(dtype == GB_F32 || dtype == GB_BF16, "gb_verify_tree: unsupported dtype %d", dtype);
    GB_REQUIRE(num_seqs < (1 << 27), "gb_verify_tree: %d requests are too many for one launch", num_seqs);
    if (num_seqs == 0) return 0;
    GB_REQUIRE(first_row && temperature && accepted && next && (n == 0 || (logits && tokens && parents && uniform && path)), "gb_verify_tree: a tensor is missing");
    VerifyArgs a = {logits, stride, draft, draft_stride, tokens, parents, first_row, uniform, temperature, path, accepted, next, n, vocab, 1};
    int blocks = VT_MAX_CLUSTER;
    while (blocks > 1 && ((long long)num_seqs * blocks > 2 * 148 || vocab < blocks * VT_SEG * VT_WARPS)) blocks /= 2;
    a.blocks = blocks;
    const int lanes = dtype == GB_F32 ? 4 : 8, per = gb_ceil_div(gb_ceil_div(vocab + lanes, VT_SEG), blocks);
    const int smem = per * (draft ? 20 : 12);
    const auto kernel = dtype == GB_F32 ? verify_tree_kernel<float> : verify_tree_kernel<__nv_bfloat16>;
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    GB_REQUIRE(e == cudaSuccess, "gb_verify_tree: %d bytes of shared memory refused: %s", smem, cudaGetErrorString(e));
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(num_seqs * blocks);
    cfg.blockDim = dim3(VT_THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    int na = 0;
    if (gb_pdl_enabled() & GB_PDL_ELEMENTWISE) {
        attr[na].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[na].val.programmaticStreamSerializationAllowed = 1;
        ++na;
    }
    if (blocks > 1) {
        attr[na].id = cudaLaunchAttributeClusterDimension;
        attr[na].val.clusterDim.x = blocks;
        attr[na].val.clusterDim.y = attr[na].val.clusterDim.z = 1;
        ++na;
    }
    cfg.attrs = attr;
    cfg.numAttrs = na;
    e = cudaLaunchKernelEx(&cfg, kernel, a);
    GB_REQUIRE(e == cudaSuccess, "gb_verify_tree: launch failed: %s", cudaGetErrorString(e));
    return gb_check_launch("gb_verify_tree");
}
