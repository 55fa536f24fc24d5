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
constexpr int VT_TABLE = 256;                           // 2^(j / 256)
constexpr int VT_ROWS = 512;                            // rows of a tree whose parents and tokens stay in shared memory

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
    double left;                       // of the leftover
    int token[2];                      // [turn] that the block found
    int warp_wrong[2][VT_WARPS];
    unsigned long long warp_best[VT_WARPS];
    double table[VT_TABLE];
    int parents[VT_ROWS], tokens[VT_ROWS];
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
__device__ __forceinline__ float vt_warp_max(float v) {                     // (not of NaN)
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}
__device__ __forceinline__ double vt_warp_sum(double v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
__device__ __forceinline__ double vt_warp_scan(double v) {                  // sums up to and with a lane's
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const double up = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += up;
    }
    return v;
}

// A float32 as a double, by its bits (0 and subnormal ones come out as numbers below 2^-126, as good as 0 beside a logit; infinities as finite ones
// beyond 2^127): the conversion proper goes through a unit that takes 16 a cycle.
__device__ __forceinline__ double vt_double(float x) {
    const unsigned b = __float_as_uint(x);
    return __hiloint2double((int)((b & 0x80000000u) | (((b & 0x7fffffffu) >> 3) + 0x38000000u)), (int)(b << 29));
}

// Weights exp((x - most) / T) of logits x <= most: 2^(k / 256) from a table, whole powers of two added to its exponent, and three terms of the exponential
// series for the rest, at most 1/512 of an octave: a relative error below (ln 2 / 512)^4 / 24 = 2^-42.7. Below e^-700 a weight is nothing.
struct VtWeight {
    const double* table;
    double heat, most;                 // 256 / (T ln 2)
    float least;
    __device__ __forceinline__ VtWeight(const double* table, double heat, float temp, float most)
        : table(table), heat(heat), most(vt_double(most)), least(fmaf(-700.0f, temp, most)) {}
    __device__ __forceinline__ double operator()(float x) const {
        constexpr double MAGIC = 6755399441055744.0;                  // 1.5 2^52: the low word of a sum with it is the nearest whole number
        constexpr double C1 = 0.0027076061740622863, C2 = 3.665565596910106e-06, C3 = 3.308302680541371e-09;      // (ln 2 / 256)^i / i!
        const double d = vt_double(fmaxf(x, least)) - most;
        const double s = fma(d, heat, MAGIC);
        const int k = __double2loint(s);
        const double r = fma(d, heat, MAGIC - s);
        const double t = table[k & (VT_TABLE - 1)];
        const double w = __hiloint2double(__double2hiint(t) + ((k >> 8) << 20), __double2loint(t));
        const double v = fma(w * r, fma(fma(C3, r, C2), r, C1), w);
        return x >= least && x > -INFINITY ? v : 0.0;
    }
};

// A lane's tokens of a segment, 16 bytes at a time: piece u * 32 + lane of the segment's. Segments begin at multiples of 16 bytes of one tensor's rows, `lead`
// numbers before the row's first; `aligned`: of this one's, too. Tokens outside the row have minus infinity.
template <typename T>
__device__ __forceinline__ void vt_load(const T* x, int lead, bool aligned, int vocab, int seg, float (&v)[VT_EACH]) {
    constexpr int N = 16 / sizeof(T);
    const int lane = threadIdx.x & 31;
    uint4 raw[VT_EACH / N];
    bool whole[VT_EACH / N];
#pragma unroll
    for (int u = 0; u < VT_EACH / N; ++u) {
        const int i = seg * VT_SEG + (u * 32 + lane) * N - lead;
        whole[u] = aligned && i >= 0 && i + N <= vocab;
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
__global__ void __launch_bounds__(VT_THREADS, 2) verify_tree_kernel(const VerifyArgs a) {
    namespace cg = cooperative_groups;
    constexpr int N = 16 / sizeof(T);
    extern __shared__ __align__(16) double vt_mem[];
    __shared__ VtShared sh;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int C = a.blocks, rank = blockIdx.x % C, seq = blockIdx.x / C, vocab = a.vocab;
    const int per = ((vocab + N + VT_SEG - 1) / VT_SEG + C - 1) / C;
    // of the block's segments: sums and largest logits of p, with drafted distributions of q, too, and the leftover's sums
    double* p_sum = vt_mem;
    double* q_sum = p_sum + per;
    double* r_sum = a.draft ? q_sum + per : q_sum;
    float* p_most = reinterpret_cast<float*>(a.draft ? r_sum + per : q_sum);
    float* q_most = p_most + per;
    for (int i = tid; i < VT_TABLE; i += VT_THREADS) sh.table[i] = exp2((double)i / VT_TABLE);
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
    const double heat = draws ? (double)VT_TABLE / ((double)temp * 0.6931471805599453) : 0.0;
    for (int i = tid; i < rows && i < VT_ROWS; i += VT_THREADS) { sh.parents[i] = a.parents[row0 + i]; sh.tokens[i] = a.tokens[row0 + i]; }
    if (rank == 0)
        for (int i = tid; i < rows; i += VT_THREADS) a.path[row0 + i] = i == 0 ? 0 : -1;
    __syncthreads();

    // The block's share of a row: largest logits and sums of its segments, and its own in `to` (for whom the cluster's barrier is still to come).
    auto scan = [&](const T* x, int lead, int lo, int hi, double* sums, float* mosts, int which, VtShare& to) {
        const bool aligned = ((uintptr_t)(x - lead) & 15) == 0;
        bool wrong = false;
        unsigned long long best = 0;
        float v[VT_EACH];
        if (lo + warp < hi) vt_load(x, lead, aligned, vocab, lo + warp, v);
        for (int seg = lo + warp; seg < hi; seg += VT_WARPS) {
            float next[VT_EACH];
            if (seg + VT_WARPS < hi) vt_load(x, lead, aligned, vocab, seg + VT_WARPS, next);
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
            if (draws) {
                most = vt_warp_max(most);
                double sum = 0.0;
                if (most > -INFINITY && most < INFINITY) {
                    const VtWeight weight(sh.table, heat, temp, most);
#pragma unroll
                    for (int i = 0; i < VT_EACH; ++i) sum += weight(v[i]);
                }
                sum = vt_warp_sum(sum);
                if (lane == 0) { sums[seg - lo] = sum; mosts[seg - lo] = most; }
            }
#pragma unroll
            for (int i = 0; i < VT_EACH; ++i) v[i] = next[i];
        }
        if (!draws) best = vt_warp_max(best);
        wrong = __any_sync(0xffffffffu, wrong);
        if (lane == 0) { sh.warp_wrong[which][warp] = wrong; sh.warp_best[warp] = best; }
        __syncthreads();
        if (warp == which) {
            wrong = __any_sync(0xffffffffu, lane < VT_WARPS && sh.warp_wrong[which][lane % VT_WARPS]);
            best = draws ? 0 : vt_warp_max(sh.warp_best[lane % VT_WARPS]);
            float most = -INFINITY;
            double sum = 0.0;
            if (draws) {
                for (int i = lane; i < hi - lo; i += 32) most = fmaxf(most, mosts[i]);
                most = vt_warp_max(most);
                if (most > -INFINITY && most < INFINITY) {
                    const VtWeight weight(sh.table, heat, temp, most);
                    for (int i = lane; i < hi - lo; i += 32) sum = fma(sums[i], weight(mosts[i]), sum);
                }
                sum = vt_warp_sum(sum);
            }
            if (lane == 0) { to.sum = sum; to.most = most; to.wrong = wrong; to.best = best; }
        }
    };
    // All blocks' shares, behind the cluster's barrier: lane b has block b's. False: no distribution.
    auto whole = [&](int turn, int which, float& most, double& sum, double& mine) -> bool {
        float m = -INFINITY;
        double s = 0.0;
        int bad = 0;
        if (lane < C) { const VtShare* o = &of(lane)->mine[turn][which]; m = o->most; s = o->sum; bad = o->wrong; }
        most = vt_warp_max(m);
        mine = 0.0;
        if (__any_sync(0xffffffffu, bad) || !(most > -INFINITY)) return false;
        mine = s * VtWeight(sh.table, heat, temp, most)(m);
        sum = vt_warp_sum(mine);
        return true;
    };
    // The token at which the sum of the weights exceeds `target`: seg_sum(i) is the sum of the block's segment i, weights(seg, w) are a lane's of one. Called by
    // warp 0 of the block in whose share it lies; `before`: the sum of the shares before; `behind`: rounding has left the target behind every weight, the last
    // one is taken.
    auto find = [&](int lo, int hi, int lead, double before, bool behind, double target, auto seg_sum, auto weights) -> int {
        int last = -1;                                 // the last segment that holds a weight
        for (int s0 = lo; s0 < hi; s0 += 32) {
            const double mine = s0 + lane < hi ? seg_sum(s0 + lane - lo) : 0.0, upto = vt_warp_scan(mine);
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
            const double upto = vt_warp_scan(mine);
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
    // The first row behind `after` that is a child of `of_row` (and holds `like`, unless that is negative); every warp for itself.
    auto next_child = [&](int of_row, int after, int like) -> int {
        for (int c0 = max(of_row, after) + 1; c0 < rows; c0 += 32) {
            const int c = c0 + lane;
            bool is = false;
            if (c < rows) {
                const int p = c < VT_ROWS ? sh.parents[c] : a.parents[row0 + c];
                is = p == of_row && (like < 0 || (c < VT_ROWS ? sh.tokens[c] : a.tokens[row0 + c]) == like);
            }
            const unsigned hit = __ballot_sync(0xffffffffu, is);
            if (hit) return c0 + __ffs(hit) - 1;
        }
        return -1;
    };

    // Every warp of every block takes the same decisions from the same numbers.
    int cur = 0, kept = 1, token = -1;
    for (int step = 0;; ++step) {                      // (a child lies behind its parent: at most `rows` steps)
        const int turn = step & 1;
        const T* x = (const T*)a.logits + (size_t)(row0 + cur) * a.stride;
        const T* y = drafted ? (const T*)a.draft + (size_t)(row0 + cur) * a.draft_stride : nullptr;
        const int lead = (int)((uintptr_t)x & 15) / (int)sizeof(T), segs = (lead + vocab + VT_SEG - 1) / VT_SEG;
        const int lo = min(rank * per, segs), hi = min(lo + per, segs);
        const bool y_aligned = drafted && ((uintptr_t)(y - lead) & 15) == 0;
        const double u = draws ? (double)a.uniform[2 * (size_t)(row0 + cur) + 1] : 0.0;
        scan(x, lead, lo, hi, p_sum, p_most, 0, sh.mine[turn][0]);
        if (drafted) scan(y, lead, lo, hi, q_sum, q_most, 1, sh.mine[turn][1]);
        cluster_sync();
        int child = -1;                                // where the walk goes on
        token = -1;
        if (!draws) {
            const unsigned long long best = vt_warp_max(lane < C ? of(lane)->mine[turn][0].best : 0ull);
            token = best ? (int)~(unsigned)best : -1;
            if (token >= 0) child = next_child(cur, cur, token);
        } else {
            float most, q_most_all = 0.f;
            double sum = 1.0, q_all = 1.0, mine, unused;
            const bool fine = whole(turn, 0, most, sum, mine), q_fine = !drafted || whole(turn, 1, q_most_all, q_all, unused);
            const VtWeight weight(sh.table, heat, temp, most), q_weight(sh.table, heat, temp, q_most_all);
            const double p_one = 1.0 / sum, q_one = 1.0 / q_all;
            double away = 0.0, left = 1.0;             // s and sum(r)
            bool from_left = false;
            auto leftover = [&](int seg, double (&w)[VT_EACH]) {
                float v[VT_EACH], z[VT_EACH];
                vt_load(x, lead, true, vocab, seg, v);
                vt_load(y, lead, y_aligned, vocab, seg, z);
#pragma unroll
                for (int i = 0; i < VT_EACH; ++i) w[i] = fmax(weight(v[i]) * p_one - away * (q_weight(z[i]) * q_one), 0.0);
            };
            if (fine && q_fine && drafted) {
                for (int c = next_child(cur, cur, -1); c >= 0; c = next_child(cur, c, -1)) {
                    const int t = c < VT_ROWS ? sh.tokens[c] : a.tokens[row0 + c];
                    if (t < 0 || t >= vocab) continue;     // (nothing that q could have given)
                    const double p = weight(gb_to_float(x[t])) * p_one, q = q_weight(gb_to_float(y[t])) * q_one, r = fmax(p - away * q, 0.0);
                    if ((double)a.uniform[2 * (size_t)(row0 + c)] * q * left < r) { child = c; break; }
                    // not taken: what is left without it
                    away += left;
                    for (int seg = lo + warp; seg < hi; seg += VT_WARPS) {
                        double w[VT_EACH], s = 0.0;
                        leftover(seg, w);
#pragma unroll
                        for (int i = 0; i < VT_EACH; ++i) s += w[i];
                        s = vt_warp_sum(s);
                        if (lane == 0) r_sum[seg - lo] = s;
                    }
                    cluster_sync();                    // (the leftover before has been read by all)
                    if (warp == 0) {
                        double s = 0.0;
                        for (int i = lane; i < hi - lo; i += 32) s += r_sum[i];
                        s = vt_warp_sum(s);
                        if (lane == 0) sh.left = s;
                    }
                    cluster_sync();
                    mine = lane < C ? of(lane)->left : 0.0;
                    left = vt_warp_sum(mine);
                    from_left = left > 0.0;
                    if (!from_left) {                  // nothing is left of r: p itself
                        whole(turn, 0, most, sum, mine);
                        break;
                    }
                }
            }
            if (fine && q_fine && child < 0) {
                // draw: the block whose share holds the target finds the token (mine: lane b has block b's share)
                const double target = u * (from_left ? left : sum), upto = vt_warp_scan(mine);
                const unsigned hit = __ballot_sync(0xffffffffu, mine > 0.0 && upto > target), some = __ballot_sync(0xffffffffu, mine > 0.0);
                const int owner = hit ? __ffs(hit) - 1 : 31 - __clz(some);
                const double before = __shfl_sync(0xffffffffu, upto - mine, max(owner, 0));
                if (owner == rank && warp == 0) {
                    auto p_seg = [&](int i) { return p_sum[i] * weight(p_most[i]); };
                    auto r_seg = [&](int i) { return r_sum[i]; };
                    auto p_weights = [&](int seg, double (&w)[VT_EACH]) {
                        float v[VT_EACH];
                        vt_load(x, lead, true, vocab, seg, v);
#pragma unroll
                        for (int i = 0; i < VT_EACH; ++i) w[i] = weight(v[i]);
                    };
                    const int found = from_left ? find(lo, hi, lead, before, !hit, target, r_seg, leftover) : find(lo, hi, lead, before, !hit, target, p_seg, p_weights);
                    if (lane == 0) sh.token[turn] = found;
                }
                cluster_sync();
                token = owner >= 0 ? of(owner)->token[turn] : -1;
                if (!drafted && token >= 0) child = next_child(cur, cur, token);
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
    const int smem = per * (draft ? 3 * 8 + 2 * 4 : 8 + 4);
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
