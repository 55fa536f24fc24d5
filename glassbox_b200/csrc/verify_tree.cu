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
// Two forms, one row's work in both (VtRow): a cluster walks with a request and reads only the rows that it reaches, one after the other (verify_walk_kernel); or
// every row is a cluster's, all at once, and leaves what would follow it, from which the walk is read off (verify_rows_kernel, verify_path_kernel). Each block of a
// cluster takes a share of the row's segments of 512 tokens, a warp a segment, and keeps their sums; they add up through distributed shared memory, and the block
// whose share holds the target finds the segment and reads it once more.
//
// What bounds it: the weights' arithmetic, 27 instructions a token and warp of which 9 are of 64 bits, and in the walk a row's trips one after the other, 6 us.
// 1 tree of 8 rows, 49,152 tokens, 8.2 us; 64 trees of 16 rows walked at T = 0.8 65 us, 512 rows of 100,003 in bfloat16 at T = 0 all at once 49 us.
#include "common.cuh"

#include <cooperative_groups.h>

constexpr int VT_MOST_WARPS = 8;
constexpr int VT_SEG = 512, VT_EACH = VT_SEG / 32;      // tokens of a segment, and of a lane
constexpr int VT_MAX_SEGS = 4097;
constexpr int VT_MAX_CLUSTER = 8;
constexpr int VT_TABLE = 64, VT_COPIES = 16;            // 2^(j / 64), j / 64 taken off its exponent's bits, for every lane of a half warp in banks of its own
constexpr double VT_NOTHING = 1e-290;                     // sums of weights below it hold none
constexpr int VT_MAX_ROWS = 8192;                        // rows of a batch whose outcomes fit shared memory
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
    int warp_wrong[2][VT_MOST_WARPS];
    unsigned long long warp_best[VT_MOST_WARPS];
    double table[VT_TABLE * VT_COPIES];
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
__device__ __forceinline__ float vt_max(float a, float b) {                 // NaN where one is
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float vt_fma_up(float a, float b, float c) {     // rounded up
    float r;
    asm("fma.rp.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
__device__ __forceinline__ float vt_warp_max(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = vt_max(v, __shfl_xor_sync(0xffffffffu, v, o));
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

// Weights exp((x - most) / T) of logits x <= most: 2^(k / 64) from a table, whole powers of two added to its exponent, and a polynomial for the rest, at most
// h = ln 2 / 128 in the exponent: 1 + r + r^2 / 2 + r^3 / 6 + r^4 / 24 with h^2 r^2 in the place of r^4, a relative error of at most h^4 / 96 = 2^-36.7. A weight
// below e^-700 is nothing (below 2^-1000; VT_NOTHING): that of a logit below `least`, which is rounded up, so that at no temperature an exponent of what is not below
// it leaves the range of numbers, and is finite, so that minus infinity has no weight at any. (One table of 256 for all lanes: 800 rows of 49,152 tokens 81 us, its banks' conflicts half of it.)
struct VtWeight {
    unsigned table;                    // (its address in shared memory: where it lies has to be known to be read there without detours)
    double heat, most;                 // 64 / (T ln 2)
    float least;
    __device__ __forceinline__ VtWeight(const double* table, double heat, float temp, float most)
        : table((unsigned)__cvta_generic_to_shared(table) + (threadIdx.x & (VT_COPIES - 1)) * 8), heat(heat), most((double)most), least(fmaxf(vt_fma_up(-700.0f, temp, most), -FLT_MAX)) {}
    __device__ __forceinline__ double operator()(float x) const {
        constexpr double MAGIC = 6755399441055744.0;                  // 1.5 2^52: the low word of a sum with it is the nearest whole number
        constexpr double C1 = 0.010830424696249145, C2 = 5.864919287185391e-05, C3 = 2.1173137155464774e-07;
        const double d = (double)fmaxf(x, least) - most;
        const double s = fma(d, heat, MAGIC);
        const int k = __double2loint(s);
        const double r = fma(d, heat, MAGIC - s);
        double t;
        asm("ld.shared.f64 %0, [%1];" : "=d"(t) : "r"(table + (unsigned)(k & (VT_TABLE - 1)) * (VT_COPIES * 8)));
        const int high = __double2hiint(t) + k * (1 << 14);               // (the entry's share of k is taken off it)
        const double w = __hiloint2double(x >= least ? high : 0, __double2loint(t));
        return fma(w * r, fma(fma(C3, r, C2), r, C1), w);
    }
};

// A lane's tokens of a segment, 16 bytes at a time: piece u * 32 + lane of the segment's. Segments begin at multiples of 16 bytes of one tensor's rows, `lead`
// numbers before the row's first; `aligned`: of this one's, too. Tokens outside the row have minus infinity.
template <typename T>
__device__ __forceinline__ void vt_load(const T* x, int lead, bool aligned, int vocab, int seg, float (&v)[VT_EACH]) {
    constexpr int N = 16 / sizeof(T);
    const int lane = threadIdx.x & 31, first = seg * VT_SEG - lead;
    if (aligned && first >= 0 && first + VT_SEG <= vocab) {
        uint4 raw[VT_EACH / N];
#pragma unroll
        for (int u = 0; u < VT_EACH / N; ++u) raw[u] = *reinterpret_cast<const uint4*>(x + first + (u * 32 + lane) * N);
#pragma unroll
        for (int u = 0; u < VT_EACH / N; ++u) {
            const unsigned w[4] = {raw[u].x, raw[u].y, raw[u].z, raw[u].w};
#pragma unroll
            for (int e = 0; e < N; ++e)
                v[u * N + e] = N == 4 ? __uint_as_float(w[e % 4]) : __uint_as_float(e & 1 ? w[(e >> 1) % 4] & 0xffff0000u : w[(e >> 1) % 4] << 16);
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < VT_EACH; ++i) {
        const int id = first + (i / N * 32 + lane) * N + i % N;
        v[i] = id >= 0 && id < vocab ? gb_to_float(x[id]) : -INFINITY;
    }
}

// What follows a row of a tree: the child that the walk goes on to, or (child -1) the token that follows it.
struct VtOutcome {
    int child, token;
};

// One row, by a cluster of C blocks (one: the block alone). Every warp of every block takes the same decisions from the same numbers.
// NW warps a block: 8 with the next segment's loads under way where few blocks have the GPU to themselves, else 4, so that many rows are in flight.
template <typename T, bool DRAFTED, int NW>
struct VtRow {
    static constexpr int VT_WARPS = NW, VT_THREADS = NW * 32;
    static constexpr bool AHEAD = NW == VT_MOST_WARPS;
    static constexpr int N = 16 / sizeof(T);
    const VerifyArgs& a;
    VtShared& sh;
    int C, rank, per, lane, warp;
    // of the block's segments: sums and largest logits of p, with drafted distributions of q, too, and the leftover's sums
    double *p_sum, *q_sum, *r_sum;
    float *p_most, *q_most;
    int row0, rows;                    // of the request
    float temp;
    bool draws;
    double heat;

    __device__ __forceinline__ VtRow(const VerifyArgs& a, VtShared& sh, double* mem, int rank) : a(a), sh(sh), C(a.blocks), rank(rank) {
        lane = threadIdx.x & 31;
        warp = threadIdx.x >> 5;
        per = ((a.vocab + N + VT_SEG - 1) / VT_SEG + C - 1) / C;
        p_sum = mem;
        q_sum = p_sum + per;
        r_sum = DRAFTED ? q_sum + per : q_sum;
        p_most = reinterpret_cast<float*>(DRAFTED ? r_sum + per : q_sum);
        q_most = p_most + per;
        static_assert(VT_THREADS % VT_TABLE == 0, "a thread has copies of one entry");
        const double power = exp2((double)(threadIdx.x % VT_TABLE) / VT_TABLE);
        const double entry = __hiloint2double(__double2hiint(power) - (int)(threadIdx.x % VT_TABLE) * (1 << 14), __double2loint(power));
        for (int i = threadIdx.x / VT_TABLE; i < VT_COPIES; i += VT_THREADS / VT_TABLE) sh.table[threadIdx.x % VT_TABLE * VT_COPIES + i] = entry;
    }
    __device__ __forceinline__ void request(int first, int count, float t) {
        row0 = first;
        rows = count;
        temp = t;
        draws = temp > 0.f;
        heat = draws ? (double)VT_TABLE / ((double)temp * 0.6931471805599453) : 0.0;
        for (int i = threadIdx.x; i < rows && i < VT_ROWS; i += VT_THREADS) { sh.parents[i] = a.parents[row0 + i]; sh.tokens[i] = a.tokens[row0 + i]; }
    }
    __device__ __forceinline__ void cluster_sync() const {
        namespace cg = cooperative_groups;
        if (C > 1) cg::this_cluster().sync(); else __syncthreads();
    }
    __device__ __forceinline__ const VtShared* of(int b) const {
        namespace cg = cooperative_groups;
        return C > 1 ? cg::this_cluster().map_shared_rank(&sh, b) : &sh;
    }

    // The block's share of a row: largest logits and sums of its segments, and its own in `to` (for whom the cluster's barrier is still to come).
    __device__ __forceinline__ void scan(const T* x, int lead, int lo, int hi, double* sums, float* mosts, int which, VtShare& to) const {
        const bool aligned = ((uintptr_t)(x - lead) & 15) == 0;
        bool wrong = false;
        float largest = -INFINITY;
        int largest_id = -1;
        float v[VT_EACH];
        if (AHEAD && lo + warp < hi) vt_load(x, lead, aligned, a.vocab, lo + warp, v);
        for (int seg = lo + warp; seg < hi; seg += VT_WARPS) {
            float next[AHEAD ? VT_EACH : 1];
            if constexpr (!AHEAD) vt_load(x, lead, aligned, a.vocab, seg, v);
            else if (seg + VT_WARPS < hi) vt_load(x, lead, aligned, a.vocab, seg + VT_WARPS, next);
            if (draws) {
                float most = -INFINITY;
#pragma unroll
                for (int i = 0; i < VT_EACH; ++i) most = vt_max(most, v[i]);
                most = vt_warp_max(most);
                wrong = wrong || !(most < INFINITY);
                double part[4] = {0.0, 0.0, 0.0, 0.0};
                if (most > -INFINITY && most < INFINITY) {
                    const VtWeight weight(sh.table, heat, temp, most);
#pragma unroll
                    for (int i = 0; i < VT_EACH; ++i) part[i & 3] += weight(v[i]);
                }
                const double sum = vt_warp_sum((part[0] + part[1]) + (part[2] + part[3]));
                if (lane == 0) { sums[seg - lo] = sum; mosts[seg - lo] = most; }
            } else {
#pragma unroll
                for (int i = 0; i < VT_EACH; ++i) {      // (a lane's ids ascend: of equal logits the first stays; NaN is passed over)
                    const int id = seg * VT_SEG + (i / N * 32 + lane) * N + i % N - lead;
                    if (v[i] > largest || (largest_id < 0 && v[i] == v[i] && (unsigned)id < (unsigned)a.vocab)) { largest = v[i]; largest_id = id; }
                }
            }
#pragma unroll
            for (int i = 0; AHEAD && i < VT_EACH; ++i) v[i] = next[i];
        }
        wrong = __any_sync(0xffffffffu, wrong);
        const unsigned long long best = draws ? 0 : vt_warp_max(largest_id >= 0 ? vt_key(largest, largest_id) : 0ull);
        if (lane == 0) { sh.warp_wrong[which][warp] = wrong; sh.warp_best[warp] = best; }
        __syncthreads();
        if (warp == which) {
            wrong = __any_sync(0xffffffffu, lane < VT_WARPS && sh.warp_wrong[which][lane % VT_WARPS]);
            const unsigned long long top = draws ? 0 : vt_warp_max(sh.warp_best[lane % VT_WARPS]);
            float most = -INFINITY;
            double sum = 0.0;
            if (draws) {
                for (int i = lane; i < hi - lo; i += 32) most = vt_max(most, mosts[i]);
                most = vt_warp_max(most);
                if (most > -INFINITY && most < INFINITY) {
                    const VtWeight weight(sh.table, heat, temp, most);
                    for (int i = lane; i < hi - lo; i += 32) sum = fma(sums[i], weight(mosts[i]), sum);
                }
                sum = vt_warp_sum(sum);
            }
            if (lane == 0) { to.sum = sum; to.most = most; to.wrong = wrong; to.best = top; }
        }
    }
    // All blocks' shares, behind the cluster's barrier: lane b has block b's. False: no distribution.
    __device__ __forceinline__ bool whole(int turn, int which, float& most, double& sum, double& mine) const {
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
    }
    // The token at which the sum of the weights exceeds `target`: seg_sum(i) is the sum of the block's segment i, weights(seg, w) are a lane's of one. Called by
    // warp 0 of the block in whose share it lies; `before`: the sum of the shares before; `behind`: rounding has left the target behind every weight, the last
    // one is taken.
    template <class Sum, class Weights>
    __device__ __forceinline__ int find(int lo, int hi, int lead, double before, bool behind, double target, Sum seg_sum, Weights weights) const {
        int last = -1;                                 // the last segment that holds a weight
        for (int s0 = lo; s0 < hi; s0 += 32) {
            const double mine = s0 + lane < hi ? seg_sum(s0 + lane - lo) : 0.0, upto = vt_warp_scan(mine);
            const unsigned some = __ballot_sync(0xffffffffu, mine > VT_NOTHING), hit = __ballot_sync(0xffffffffu, mine > VT_NOTHING && !behind && before + upto > target);
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
        double w[VT_EACH], mine[VT_EACH / N], upto[VT_EACH / N];
        weights(last, w);
#pragma unroll
        for (int u = 0; u < VT_EACH / N; ++u) {
            mine[u] = 0.0;
#pragma unroll
            for (int e = 0; e < N; ++e) mine[u] += w[u * N + e];
            upto[u] = vt_warp_scan(mine[u]);
        }
        int token = -1;
#pragma unroll
        for (int u = 0; u < VT_EACH / N; ++u) {
            double sum = before + upto[u] - mine[u];
            int found = -1, held = -1;                 // where the sum passes the target, and the lane's last weight
#pragma unroll
            for (int e = 0; e < N; ++e) {
                const int id = last * VT_SEG + (u * 32 + lane) * N + e - lead;
                sum += w[u * N + e];
                if (w[u * N + e] > VT_NOTHING) {
                    held = id;
                    if (found < 0 && sum > target && !behind) found = id;
                }
            }
            const unsigned hit = __ballot_sync(0xffffffffu, found >= 0), some = __ballot_sync(0xffffffffu, held >= 0);
            if (hit) return __shfl_sync(0xffffffffu, found, __ffs(hit) - 1);
            if (some) token = __shfl_sync(0xffffffffu, held, 31 - __clz(some));
            before += __shfl_sync(0xffffffffu, upto[u], 31);
        }
        return token;
    }
    // The first row behind `after` that is a child of `of_row` (and holds `like`, unless that is negative); every warp for itself.
    __device__ __forceinline__ int next_child(int of_row, int after, int like) const {
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
    }

    // turn: 0 and 1 from call to call, so that what blocks still read of one is not written by the next.
    __device__ __forceinline__ VtOutcome outcome(int cur, int turn) const {
        const int vocab = a.vocab;
        const bool drafted = DRAFTED && draws && next_child(cur, cur, -1) >= 0;      // (a row without children has no q)
        const T* x = (const T*)a.logits + (size_t)(row0 + cur) * a.stride;
        const T* y = drafted ? (const T*)a.draft + (size_t)(row0 + cur) * a.draft_stride : nullptr;
        const int lead = (int)((uintptr_t)x & 15) / (int)sizeof(T), segs = (lead + vocab + VT_SEG - 1) / VT_SEG;
        const int lo = min(rank * per, segs), hi = min(lo + per, segs);
        const bool y_aligned = drafted && ((uintptr_t)(y - lead) & 15) == 0;
        const double u = draws ? (double)a.uniform[2 * (size_t)(row0 + cur) + 1] : 0.0;
        scan(x, lead, lo, hi, p_sum, p_most, 0, sh.mine[turn][0]);
        if (drafted) scan(y, lead, lo, hi, q_sum, q_most, 1, sh.mine[turn][1]);
        cluster_sync();
        if (!draws) {
            const unsigned long long best = vt_warp_max(lane < C ? of(lane)->mine[turn][0].best : 0ull);
            const int token = best ? (int)~(unsigned)best : -1;
            return {token >= 0 ? next_child(cur, cur, token) : -1, token};
        }
        float most, q_most_all = 0.f;
        double sum = 1.0, q_all = 1.0, mine, unused;
        if (!whole(turn, 0, most, sum, mine)) return {-1, -1};
        if (drafted && !whole(turn, 1, q_most_all, q_all, unused)) return {-1, -1};
        const VtWeight weight(sh.table, heat, temp, most), q_weight(sh.table, heat, temp, q_most_all);
        const double p_one = 1.0 / sum, q_one = 1.0 / q_all;
        double away = 0.0, left = 1.0;                 // s and sum(r)
        bool from_left = false;
        auto leftover = [&](int seg, double (&w)[VT_EACH]) {
            float v[VT_EACH], z[VT_EACH];
            vt_load(x, lead, true, vocab, seg, v);
            vt_load(y, lead, y_aligned, vocab, seg, z);
#pragma unroll
            for (int i = 0; i < VT_EACH; ++i) w[i] = fmax(weight(v[i]) * p_one - away * (q_weight(z[i]) * q_one), 0.0);
        };
        if (drafted) {
            for (int c = next_child(cur, cur, -1); c >= 0; c = next_child(cur, c, -1)) {
                const int t = c < VT_ROWS ? sh.tokens[c] : a.tokens[row0 + c];
                if (t < 0 || t >= vocab) continue;     // (nothing that q could have given)
                const double p = weight(gb_to_float(x[t])) * p_one, q = q_weight(gb_to_float(y[t])) * q_one, r = fmax(p - away * q, 0.0);
                if (r > VT_NOTHING && (double)a.uniform[2 * (size_t)(row0 + c)] * q * left < r) return {c, t};
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
                cluster_sync();                        // (the leftover before has been read by all)
                if (warp == 0) {
                    double s = 0.0;
                    for (int i = lane; i < hi - lo; i += 32) s += r_sum[i];
                    s = vt_warp_sum(s);
                    if (lane == 0) sh.left = s;
                }
                cluster_sync();
                mine = lane < C ? of(lane)->left : 0.0;
                left = vt_warp_sum(mine);
                from_left = left > VT_NOTHING;
                if (!from_left) {                      // nothing is left of r: p itself
                    whole(turn, 0, most, sum, mine);
                    break;
                }
            }
        }
        // draw: the block whose share holds the target finds the token (mine: lane b has block b's share)
        const double target = u * (from_left ? left : sum), upto = vt_warp_scan(mine);
        const unsigned hit = __ballot_sync(0xffffffffu, mine > VT_NOTHING && upto > target), some = __ballot_sync(0xffffffffu, mine > VT_NOTHING);
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
            int found;
            if (DRAFTED && from_left) found = find(lo, hi, lead, before, !hit, target, r_seg, leftover);
            else found = find(lo, hi, lead, before, !hit, target, p_seg, p_weights);
            if (lane == 0) sh.token[turn] = found;
        }
        cluster_sync();
        const int token = owner >= 0 ? of(owner)->token[turn] : -1;
        return {!drafted && token >= 0 ? next_child(cur, cur, token) : -1, token};
    }
};

// A cluster walks with a request: only the rows that it reaches are read.
template <typename T, bool DRAFTED, int NW>
__global__ void __launch_bounds__(NW * 32, 16 / NW) verify_walk_kernel(const VerifyArgs a) {
    extern __shared__ __align__(16) double vt_mem[];
    __shared__ VtShared sh;
    const int rank = blockIdx.x % a.blocks, seq = blockIdx.x / a.blocks;
    VtRow<T, DRAFTED, NW> row(a, sh, vt_mem, rank);
    gb_pdl_launch_dependents();
    gb_pdl_wait();
    const int row0 = a.first_row[seq], rows = a.first_row[seq + 1] - row0;
    if (rows <= 0 || row0 < 0 || row0 > a.n - rows) {  // (the same in all blocks of a cluster)
        if (rank == 0 && threadIdx.x == 0) { a.accepted[seq] = 0; a.next[seq] = -1; }
        return;
    }
    row.request(row0, rows, a.temperature[seq]);
    if (rank == 0)
        for (int i = threadIdx.x; i < rows; i += NW * 32) a.path[row0 + i] = i == 0 ? 0 : -1;
    __syncthreads();
    int cur = 0, kept = 1;
    for (int step = 0;; ++step) {                      // (a child lies behind its parent: at most `rows` steps)
        const VtOutcome o = row.outcome(cur, step & 1);
        if (o.child < 0) {
            if (rank == 0 && threadIdx.x == 0) { a.accepted[seq] = kept; a.next[seq] = o.token; }
            break;
        }
        cur = o.child;
        if (rank == 0 && threadIdx.x == 0) a.path[row0 + kept] = cur;
        ++kept;
    }
    row.cluster_sync();                                // (shared memory is read until here)
}

// Every row's outcome at once, a cluster a row: the child, or -2 - token, in the row's place of `path`, from which verify_path_kernel walks.
template <typename T, bool DRAFTED, int NW>
__global__ void __launch_bounds__(NW * 32, (DRAFTED ? 20 : NW == VT_MOST_WARPS ? 24 : 32) / NW) verify_rows_kernel(const VerifyArgs a, int num_seqs) {
    extern __shared__ __align__(16) double vt_mem[];
    __shared__ VtShared sh;
    const int rank = blockIdx.x % a.blocks, r = blockIdx.x / a.blocks, lane = threadIdx.x & 31;
    VtRow<T, DRAFTED, NW> row(a, sh, vt_mem, rank);
    gb_pdl_launch_dependents();
    gb_pdl_wait();
    int seq = -1;                                      // the last request that begins at the row or before it and is not empty
    for (int s0 = 0; s0 < num_seqs; s0 += 32) {
        const int s = s0 + lane, first = s < num_seqs ? a.first_row[s] : 0, next = s < num_seqs ? a.first_row[s + 1] : 0;
        const unsigned hit = __ballot_sync(0xffffffffu, s < num_seqs && first >= 0 && first <= r && r < next && next <= a.n);
        if (hit) { seq = s0 + __ffs(hit) - 1; break; }
    }
    if (seq < 0) return;                               // (a row of no request)
    const int row0 = a.first_row[seq];
    row.request(row0, a.first_row[seq + 1] - row0, a.temperature[seq]);
    __syncthreads();
    const VtOutcome o = row.outcome(r - row0, 0);
    if (rank == 0 && threadIdx.x == 0) a.path[r] = o.child >= 0 ? o.child : -2 - o.token;
    row.cluster_sync();                                // (shared memory is read until here)
}

// The walk over the rows' outcomes: a warp a request.
__global__ void __launch_bounds__(32) verify_path_kernel(const VerifyArgs a) {
    extern __shared__ int vt_next[];
    const int seq = blockIdx.x, lane = threadIdx.x;
    gb_pdl_launch_dependents();
    gb_pdl_wait();
    const int row0 = a.first_row[seq], rows = a.first_row[seq + 1] - row0;
    if (rows <= 0 || row0 < 0 || row0 > a.n - rows) {
        if (lane == 0) { a.accepted[seq] = 0; a.next[seq] = -1; }
        return;
    }
    for (int i = lane; i < rows; i += 32) vt_next[i] = a.path[row0 + i];
    __syncwarp();
    int kept = 0;
    for (int cur = 0;;) {
        if (lane == 0) a.path[row0 + kept] = cur;
        ++kept;
        const int o = vt_next[cur];
        if (o <= cur || o >= rows) {                   // (a child lies behind its row)
            if (lane == 0) { a.accepted[seq] = kept; a.next[seq] = o < 0 ? -2 - o : -1; }
            break;
        }
        cur = o;
    }
    for (int i = kept + lane; i < rows; i += 32) a.path[row0 + i] = -1;
}

template <typename T, bool DRAFTED, int NW>
static int vt_launch(VerifyArgs a, int num_seqs, bool walk, int groups, int blocks, cudaStream_t stream) {
    a.blocks = blocks;
    const int per = gb_ceil_div(gb_ceil_div(a.vocab + 16 / (int)sizeof(T), VT_SEG), blocks), smem = per * (DRAFTED ? 3 * 8 + 2 * 4 : 8 + 4);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(groups * blocks));
    cfg.blockDim = dim3(NW * 32);
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
    cudaError_t e = walk ? cudaFuncSetAttribute(verify_walk_kernel<T, DRAFTED, NW>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem)
                         : cudaFuncSetAttribute(verify_rows_kernel<T, DRAFTED, NW>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    GB_REQUIRE(e == cudaSuccess, "gb_verify_tree: %d bytes of shared memory refused: %s", smem, cudaGetErrorString(e));
    e = walk ? cudaLaunchKernelEx(&cfg, verify_walk_kernel<T, DRAFTED, NW>, a) : cudaLaunchKernelEx(&cfg, verify_rows_kernel<T, DRAFTED, NW>, a, num_seqs);
    GB_REQUIRE(e == cudaSuccess, "gb_verify_tree: launch failed: %s", cudaGetErrorString(e));
    return 0;
}

template <typename T, bool DRAFTED>
static int vt_dispatch(const VerifyArgs& a, int num_seqs, bool walk, cudaStream_t stream) {
    // Blocks that share a row while all find room at once, eight of four warps a multiprocessor, two segments a warp at least: 388 rows of 100,003 bfloat16 in
    // clusters of 1 / 2 / 4 70 / 49 / 53 us, 768 of 49,152 float32 64 / 66 / 76. Up to two blocks a multiprocessor have eight warps: 8 rows of
    // 49,152 12.3 us and with four warps 14.4, 1 of 128,256 12.4 and 16.4; 64 rows 22.6 and 16.5.
    const int groups = walk ? num_seqs : a.n;
    int blocks = VT_MAX_CLUSTER;
    while (blocks > 1 && ((long long)groups * blocks > 8 * 148 || a.vocab < blocks * VT_SEG * VT_MOST_WARPS)) blocks /= 2;
    if ((long long)groups * blocks <= 2 * 148) return vt_launch<T, DRAFTED, VT_MOST_WARPS>(a, num_seqs, walk, groups, blocks, stream);
    return vt_launch<T, DRAFTED, VT_MOST_WARPS / 2>(a, num_seqs, walk, groups, blocks, stream);
}

// logits, draft: [n, vocab] of one type, rows `stride` numbers apart (draft: or none). Everything else as above; path [n], accepted and next [requests]. walk: as
// verify_walk_kernel, else all rows at once; no request has more than max_rows rows then.
GB_EXPORT int gb_verify_tree(const void* logits, int dtype, long long stride, const void* draft, long long draft_stride, const int* tokens, const int* parents,
                             const int* first_row, const float* uniform, const float* temperature, int* path, int* accepted, int* next, int n, int num_seqs,
                             int vocab, int walk, cudaStream_t stream) {
    GB_REQUIRE(n >= 0 && num_seqs >= 0 && vocab > 0 && (n <= 1 || stride >= vocab) && (draft == nullptr || n <= 1 || draft_stride >= vocab), "gb_verify_tree: bad sizes n=%d vocab=%d", n, vocab);
    GB_REQUIRE(vocab <= (VT_MAX_SEGS - 1) * VT_SEG, "gb_verify_tree: a vocabulary of %d is not built (%d)", vocab, (VT_MAX_SEGS - 1) * VT_SEG);
    GB_REQUIRE(dtype == GB_F32 || dtype == GB_BF16, "gb_verify_tree: unsupported dtype %d", dtype);
    GB_REQUIRE(num_seqs < (1 << 27) && n < (1 << 27), "gb_verify_tree: %d requests, %d rows are too many for one launch", num_seqs, n);
    if (num_seqs == 0) return 0;
    GB_REQUIRE(first_row && temperature && accepted && next && (n == 0 || (logits && tokens && parents && uniform && path)), "gb_verify_tree: a tensor is missing");
    const VerifyArgs a = {logits, stride, draft, draft_stride, tokens, parents, first_row, uniform, temperature, path, accepted, next, n, vocab, 1};
    if (n > VT_MAX_ROWS || n == 0) walk = 1;           // (a request's outcomes fit shared memory)
    const int rc = dtype == GB_F32 ? (draft ? vt_dispatch<float, true>(a, num_seqs, walk, stream) : vt_dispatch<float, false>(a, num_seqs, walk, stream))
                                   : (draft ? vt_dispatch<__nv_bfloat16, true>(a, num_seqs, walk, stream) : vt_dispatch<__nv_bfloat16, false>(a, num_seqs, walk, stream));
    if (rc) return rc;
    if (!walk) {
        const cudaError_t e = gb_launch(GB_PDL_ELEMENTWISE, verify_path_kernel, dim3(num_seqs), dim3(32), n * sizeof(int), stream, a);
        GB_REQUIRE(e == cudaSuccess, "gb_verify_tree: launch failed: %s", cudaGetErrorString(e));
    }
    return gb_check_launch("gb_verify_tree");
}
