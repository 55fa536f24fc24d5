// Decode attention over a cache in 4 bits (layout: kv4.cuh) in bfloat16 on the tensor cores.
//
// One block = one row, up to eight query heads of one kv head, one share of the row's keys; its warps take the share's tiles of 16 keys in
// turn. A tile is one contiguous piece of the pool for keys and one for values, and each warp has a ring of STAGES of both in shared
// memory that one lane keeps full with bulk copies: nothing but the lane's two instructions per tile is spent on addresses, and the copies that a
// multiprocessor has in flight (16 warps x 3 tiles x 18 hd bytes) are several times what the memory's latency asks for.
//
// Codes become operands of mma.sync m16n8k16 without being scaled: a code u in four bits, put under 0x4300, is the bfloat16 128 + u.
//   * S = Q K^T, the heads as the 16 rows of A (eight of them zero), 8 keys a column tile: the sums of a group of 32 channels come out as
//     sum q (128 + u), from which 136 sum q is subtracted (u = s + 8; both are float32 sums of exact products, so this costs 5 of their
//     24 bits), and the key's scale is applied to what is left: one multiplication a key, head and group instead of one a number.
//   * O^T = V^T P^T, 16 channels of a group as the rows, the heads as columns: p times the value's scale is rounded to bfloat16 (the
//     only rounding of the kernel besides the result's: half a step is 2^-9 of the weight, as every kernel here that multiplies weights on
//     the tensor cores), codes less 136 are whole numbers that bfloat16 holds. A thread's sums of S are the B operand of this product as they lie.
//     (Values cannot keep their 128 + 8: the sum over thousands of keys would be 136 sum p against results near zero.)
// The reference that is subtracted from scores rises only when one exceeds it by 2^8 (weights up to 256 cost the float32 sums nothing), so that
// the sums of O are hardly ever rescaled.
// The warps of a block add up in shared memory, the blocks of a row in a cluster (each adds up some of the heads from all of the
// others' shared memory); where a row has more shares than a cluster has blocks, the clusters' results go through `parts` and
// kv4_merge_kernel. Nothing is left behind for the next call.
#include <atomic>

#include "kv4_attention.cuh"
#include "tcgen05.cuh"

constexpr int KV4M_WARPS = 4;
constexpr int KV4M_HEADS = 8;      // query heads of a block

__device__ __forceinline__ void kv4_mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void kv4_bulk(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}
__device__ __forceinline__ float kv4_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// nibble i and nibble i + 4 of w as two bfloat16 128 + u
__device__ __forceinline__ uint32_t kv4_up(uint32_t w, int i) {
    uint32_t r;
    asm("lop3.b32 %0, %1, 0x000f000f, 0x43004300, 0xea;" : "=r"(r) : "r"(w >> (4 * i)));      // (a & b) | c
    return r;
}
__device__ __forceinline__ uint32_t kv4_down(uint32_t v) {                                        // 128 + u -> s, twice
    const uint32_t c = 0x43084308u;
    const __nv_bfloat162 r = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&v), *reinterpret_cast<const __nv_bfloat162*>(&c));
    return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t kv4_pack(float lo, float hi) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ float kv4_bf16(const uint32_t* words, int i) {       // number i of packed bfloat16
    return i & 1 ? __uint_as_float(words[i >> 1] & 0xffff0000u) : __uint_as_float(words[i >> 1] << 16);
}

// W consecutive 32-bit words from shared memory (aligned to all of them, up to 16 bytes)
template <int W> __device__ __forceinline__ void kv4_words(const unsigned char* p, uint32_t (&w)[W]) {
    if constexpr (W % 4 == 0) {
#pragma unroll
        for (int i = 0; i < W; i += 4) {
            const uint4 v = *reinterpret_cast<const uint4*>(p + 4 * i);
            w[i] = v.x; w[i + 1] = v.y; w[i + 2] = v.z; w[i + 3] = v.w;
        }
    } else if constexpr (W == 2) {
        const uint2 v = *reinterpret_cast<const uint2*>(p);
        w[0] = v.x; w[1] = v.y;
    } else {
#pragma unroll
        for (int i = 0; i < W; ++i) w[i] = *reinterpret_cast<const uint32_t*>(p + 4 * i);
    }
}

template <int HD> struct Kv4Geometry {
    static constexpr int G = HD / KV4_GROUP;
    static constexpr int TILE = kv4_tile_bytes(HD);                       // bytes of a tile of keys, or of values
    static constexpr int STAGES = HD <= 64 ? 6 : HD <= 128 ? 4 : 3;
    static constexpr int RING = STAGES * 2 * TILE;                        // of a warp
    static constexpr int PART = KV4M_HEADS * (HD + 2) * 4;                // bytes of a warp's, or the block's, result: maxima, sums, rows
    static constexpr int SMEM = KV4M_WARPS * RING > (KV4M_WARPS + 1) * PART ? KV4M_WARPS * RING : (KV4M_WARPS + 1) * PART;
};

template <int HD>
__global__ void __launch_bounds__(KV4M_WARPS * 32) kv4_decode_mma_kernel(const Kv4AttnArgs a, const int cluster) {
    using Geo = Kv4Geometry<HD>;
    constexpr int G = Geo::G, STAGES = Geo::STAGES, TILE = Geo::TILE;
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ __align__(8) uint64_t full[KV4M_WARPS][STAGES];
    __shared__ int gave_up;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int group = a.nh / a.nkv, chunks = (group + KV4M_HEADS - 1) / KV4M_HEADS;
    const int kvh = blockIdx.y / chunks, head0 = kvh * group + (blockIdx.y % chunks) * KV4M_HEADS;
    const int heads = min(KV4M_HEADS, (kvh + 1) * group - head0), row = blockIdx.z, split = blockIdx.x;

    if (threadIdx.x == 0) gave_up = 0;
    if (lane < STAGES) mbar_init(&full[warp][lane], 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    __syncthreads();
    gb_pdl_wait();
    gb_pdl_launch_dependents();

    int pos = a.positions[row];
    if (pos >= 0 && pos / a.page_size >= a.max_pages) {   // a position the block table does not reach: reported, the row reads nothing
        if (threadIdx.x == 0 && blockIdx.x == 0 && blockIdx.y == 0) atomicOr(a.status, GB_STATUS_BAD_POSITION);
        pos = -1;
    }
    const int first = gb_first_key(pos, a.window), tile0 = first / KV4_TILE, tiles = pos < 0 ? 0 : pos / KV4_TILE - tile0 + 1;
    const int begin = tile0 + kv4_share(tiles, split, gridDim.x), end = tile0 + kv4_share(tiles, split + 1, gridDim.x);
    const int mine = end - begin > warp ? (end - begin - warp + KV4M_WARPS - 1) / KV4M_WARPS : 0;      // tiles begin + warp + KV4M_WARPS * i
    const int* table = a.block_tables + (size_t)(pos < 0 ? 0 : a.row_seq[row]) * a.max_pages;
    const int per_page = a.page_size / KV4_TILE;
    unsigned char* ring = smem + warp * Geo::RING;

    // Where the tiles of this warp lie, 32 tiles at a time, one a lane: the tile's number in the pool, or -1 for a page that is missing.
    long long place[2];
    auto look = [&](int i) -> long long {
        if (i >= mine) return -1;
        const int tile = begin + warp + KV4M_WARPS * i, pi = tile / per_page;
        const long long page = table[pi];
        if (page < 0 || page >= a.num_pages) {
            atomicOr(a.status, GB_STATUS_BAD_SLOT);
            return -1;
        }
        return (page * a.nkv + kvh) * per_page + tile % per_page;
    };
    place[0] = look(lane);
    place[1] = look(32 + lane);
    auto issue = [&](int i) {       // (all lanes; i < mine)
        const long long at = __shfl_sync(0xffffffffu, (i >> 5) & 1 ? place[1] : place[0], i & 31);
        if (at >= 0 && lane == 0) {
            const int s = i % STAGES;
            const uint32_t bar = smem_u32(&full[warp][s]), dst = smem_u32(ring + s * 2 * TILE);
            mbar_expect_tx(&full[warp][s], 2 * TILE);
            kv4_bulk(dst, a.kcache + at * TILE, TILE, bar);
            kv4_bulk(dst + TILE, a.vcache + at * TILE, TILE, bar);
        }
        return at >= 0;
    };
    unsigned there = 0, parity = 0;          // per stage: a copy has been asked for; the phase its next completion ends
#pragma unroll
    for (int i = 0; i < STAGES - 1; ++i)
        if (i < mine && issue(i)) there |= 1u << i;

    // Q as the A operand: row g is head head0 + g; the two k16 steps of a group take channels 8 t + {0, 4, 1, 5} and {2, 6, 3, 7} of it
    // at this thread's places, as a word of eight codes yields them.
    uint32_t qf[G][4];
    float qsum[G];
    {
        const __nv_bfloat16* q = (const __nv_bfloat16*)a.q + (size_t)row * a.q_stride + (size_t)(head0 + g) * HD + 8 * t;
        const bool wide = (((uintptr_t)a.q | (uintptr_t)(a.q_stride * 2)) & 15) == 0;
#pragma unroll
        for (int i = 0; i < G; ++i) {
            uint32_t w[4] = {0, 0, 0, 0};
            if (g < heads) {
                if (wide) {
                    const uint4 v = *reinterpret_cast<const uint4*>(q + 32 * i);
                    w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
                } else {
                    const unsigned short* p = reinterpret_cast<const unsigned short*>(q + 32 * i);
#pragma unroll
                    for (int j = 0; j < 4; ++j) w[j] = p[2 * j] | (uint32_t)p[2 * j + 1] << 16;
                }
            }
            qf[i][0] = __byte_perm(w[0], w[2], 0x5410);
            qf[i][1] = __byte_perm(w[0], w[2], 0x7632);
            qf[i][2] = __byte_perm(w[1], w[3], 0x5410);
            qf[i][3] = __byte_perm(w[1], w[3], 0x7632);
            float sum = 0.f;
#pragma unroll
            for (int j = 0; j < 8; ++j) sum += kv4_bf16(w, j);
            sum += __shfl_xor_sync(0xffffffffu, sum, 1);
            sum += __shfl_xor_sync(0xffffffffu, sum, 2);
            qsum[i] = -136.f * sum;
        }
    }

    float m = KV4_NEG_BIG, l = 0.f;          // of head g; l: this thread's keys
    float o[G][2][4];                        // [group][pair of channels]: channel 32 i + 4 g + 2 j (and + 1 in [2], [3]) of heads 2 t, 2 t + 1
#pragma unroll
    for (int i = 0; i < G; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[i][j][e] = 0.f;

    bool alive = true;
    for (int i = 0; i < mine; ++i) {
        if ((i & 31) == 0 && i > 0) {        // the next 32, while these are worked on
            const long long next = look(i + 32 + lane);
            if (i & 32) place[0] = next;
            else place[1] = next;
        }
        const int s = i % STAGES;
        {
            const int ahead = i + STAGES - 1, sa = ahead % STAGES;
            there &= ~(1u << sa);            // (that stage's tile was read an iteration ago, by all lanes: the barrier at the end of it)
            if (ahead < mine && issue(ahead)) there |= 1u << sa;
        }
        if (!(there >> s & 1)) continue;     // a missing page: its keys are not there
        alive = mbar_wait_warp(&full[warp][s], parity >> s & 1, &gave_up, a.status);
        if (!alive) break;
        parity ^= 1u << s;
        const unsigned char* kt = ring + s * 2 * TILE;
        const unsigned char* vt = kt + TILE;
        const int key0 = (begin + warp + KV4M_WARPS * i) * KV4_TILE;

        // ---- scores of keys 8 j + 2 t, 8 j + 2 t + 1 for head g
        float sc[2][2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            uint32_t w[G], d[G];
            kv4_words<G>(kt + (8 * j + g) * (HD / 2) + t * G * 4, w);
            kv4_words<G>(kt + 8 * HD + (8 * j + 2 * t) * G * 2, d);      // scales of the two keys: G and G of them
            sc[j][0] = sc[j][1] = 0.f;
#pragma unroll
            for (int k = 0; k < G; ++k) {
                float c[4] = {0.f, 0.f, 0.f, 0.f};
                kv4_mma(c, qf[k][0], 0u, qf[k][1], 0u, kv4_up(w[k], 0), kv4_up(w[k], 1));
                kv4_mma(c, qf[k][2], 0u, qf[k][3], 0u, kv4_up(w[k], 2), kv4_up(w[k], 3));
                sc[j][0] = fmaf(kv4_bf16(d, k), c[0] + qsum[k], sc[j][0]);
                sc[j][1] = fmaf(kv4_bf16(d, G + k), c[1] + qsum[k], sc[j][1]);
            }
        }
        // ---- weights
        const bool edge = key0 < first || key0 + KV4_TILE - 1 > pos;
        float most = KV4_NEG_BIG;
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                sc[j][e] *= a.scale;
                if (edge) {
                    const int key = key0 + 8 * j + 2 * t + e;
                    if (key < first || key > pos) sc[j][e] = -INFINITY;
                }
                most = fmaxf(most, sc[j][e]);
            }
        if (__any_sync(0xffffffffu, most > m + 8.f)) {
            most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
            most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
            const float m_new = fmaxf(m, most), corr = kv4_exp2(m - m_new);
            m = m_new;
            l *= corr;
            const float c0 = __shfl_sync(0xffffffffu, corr, 8 * t), c1 = __shfl_sync(0xffffffffu, corr, 8 * t + 4);
#pragma unroll
            for (int k = 0; k < G; ++k)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    o[k][j][0] *= c0; o[k][j][1] *= c1; o[k][j][2] *= c0; o[k][j][3] *= c1;
                }
        }
        float p[2][2];
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                p[j][e] = kv4_exp2(sc[j][e] - m);
                l += p[j][e];
            }
        // ---- output: weights times the values' scales as the B operand, codes of keys 2 t, 2 t + 1, 2 t + 8, 2 t + 9 as the A operand
        uint32_t b[2][G];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            uint32_t d[G];
            kv4_words<G>(vt + 8 * HD + (8 * j + 2 * t) * G * 2, d);
#pragma unroll
            for (int k = 0; k < G; ++k) {
                float x0 = p[j][0] * kv4_bf16(d, k), x1 = p[j][1] * kv4_bf16(d, G + k);
                if (edge) {                  // (the scale of a token that is not in sight may be anything)
                    const int key = key0 + 8 * j + 2 * t;
                    if (key < first || key > pos) x0 = 0.f;
                    if (key + 1 < first || key + 1 > pos) x1 = 0.f;
                }
                b[j][k] = kv4_pack(x0, x1);
            }
        }
        const unsigned char* vr = vt + 2 * t * (HD / 2) + g * G * 2;
        if constexpr (G % 2 == 0) {
            uint32_t w[4][G / 2];
            kv4_words<G / 2>(vr, w[0]);
            kv4_words<G / 2>(vr + HD / 2, w[1]);
            kv4_words<G / 2>(vr + 8 * (HD / 2), w[2]);
            kv4_words<G / 2>(vr + 9 * (HD / 2), w[3]);
#pragma unroll
            for (int k = 0; k < G; ++k) {
                const uint32_t lo = __byte_perm(w[0][k / 2], w[1][k / 2], k & 1 ? 0x7632 : 0x5410);
                const uint32_t hi = __byte_perm(w[2][k / 2], w[3][k / 2], k & 1 ? 0x7632 : 0x5410);
#pragma unroll
                for (int j = 0; j < 2; ++j)
                    kv4_mma(o[k][j], kv4_down(kv4_up(lo, 2 * j)), kv4_down(kv4_up(lo, 2 * j + 1)), kv4_down(kv4_up(hi, 2 * j)),
                            kv4_down(kv4_up(hi, 2 * j + 1)), b[0][k], b[1][k]);
            }
        } else {
#pragma unroll
            for (int k = 0; k < G; ++k) {
                const unsigned short* h = reinterpret_cast<const unsigned short*>(vr) + k;
                const uint32_t lo = h[0] | (uint32_t)h[HD / 4] << 16, hi = h[8 * (HD / 4)] | (uint32_t)h[9 * (HD / 4)] << 16;
#pragma unroll
                for (int j = 0; j < 2; ++j)
                    kv4_mma(o[k][j], kv4_down(kv4_up(lo, 2 * j)), kv4_down(kv4_up(lo, 2 * j + 1)), kv4_down(kv4_up(hi, 2 * j)),
                            kv4_down(kv4_up(hi, 2 * j + 1)), b[0][k], b[1][k]);
            }
        }
        __syncwarp();                        // every lane has read this stage
    }
    if (!alive)                              // a wait ran out: the copies still under way end before their memory is used again
        for (int s = 0; s < STAGES; ++s)
            if (there >> s & 1)
                for (int spin = 0; spin < 1000 && !mbar_try_wait(&full[warp][s], parity >> s & 1); ++spin) {}

    // ---- the warps' results: maxima [8], sums [8], rows [8][HD] each
    l += __shfl_xor_sync(0xffffffffu, l, 1);
    l += __shfl_xor_sync(0xffffffffu, l, 2);
    __syncthreads();
    float* parts = reinterpret_cast<float*>(smem);
    constexpr int PART = Geo::PART / 4;
    {
        float* w = parts + warp * PART;
        if (t == 0) { w[g] = m; w[8 + g] = l; }
#pragma unroll
        for (int k = 0; k < G; ++k)
#pragma unroll
            for (int h = 0; h < 2; ++h)
                *reinterpret_cast<float4*>(w + 16 + (2 * t + h) * HD + 32 * k + 4 * g) = make_float4(o[k][0][h], o[k][0][2 + h], o[k][1][h], o[k][1][2 + h]);
    }
    __syncthreads();
    float* block = parts + KV4M_WARPS * PART;
    for (int i = threadIdx.x; i < heads * (HD / 4); i += KV4M_WARPS * 32) {
        const int h = i / (HD / 4), c = i % (HD / 4) * 4;
        float most = KV4_NEG_BIG, sum = 0.f;
        float4 r = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < KV4M_WARPS; ++w) most = fmaxf(most, parts[w * PART + h]);
#pragma unroll
        for (int w = 0; w < KV4M_WARPS; ++w) {
            const float f = kv4_exp2(parts[w * PART + h] - most);
            const float4 v = *reinterpret_cast<const float4*>(parts + w * PART + 16 + h * HD + c);
            sum = fmaf(parts[w * PART + 8 + h], f, sum);
            r.x = fmaf(v.x, f, r.x); r.y = fmaf(v.y, f, r.y); r.z = fmaf(v.z, f, r.z); r.w = fmaf(v.w, f, r.w);
        }
        if (c == 0) { block[h] = most; block[8 + h] = sum; }
        *reinterpret_cast<float4*>(block + 16 + h * HD + c) = r;
    }
    // ---- the blocks of a cluster: each adds up every cluster-th piece from all of them, in their order
    if (cluster > 1) {
        asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    } else {
        __syncthreads();
    }
    const int rank = cluster > 1 ? split % cluster : 0, outer = gridDim.x / cluster;
    const uint32_t own = smem_u32(block);
    auto peer = [&](int r, int at) -> uint32_t {
        uint32_t p;
        asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(p) : "r"(own + 4 * at), "r"(r));
        return p;
    };
    auto get = [&](int r, int at) -> float {
        if (cluster == 1) return block[at];
        float v;
        asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(peer(r, at)));
        return v;
    };
    auto get4 = [&](int r, int at) -> float4 {
        if (cluster == 1) return *reinterpret_cast<const float4*>(block + at);
        float4 v;
        asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(peer(r, at)));
        return v;
    };
    for (int i = rank * KV4M_WARPS * 32 + threadIdx.x; i < heads * (HD / 4); i += cluster * KV4M_WARPS * 32) {
        const int h = i / (HD / 4), c = i % (HD / 4) * 4;
        float most = KV4_NEG_BIG, sum = 0.f;
        float4 r = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int w = 0; w < cluster; ++w) most = fmaxf(most, get(w, h));
        for (int w = 0; w < cluster; ++w) {
            const float f = kv4_exp2(get(w, h) - most);
            const float4 v = get4(w, 16 + h * HD + c);
            sum = fmaf(get(w, 8 + h), f, sum);
            r.x = fmaf(v.x, f, r.x); r.y = fmaf(v.y, f, r.y); r.z = fmaf(v.z, f, r.z); r.w = fmaf(v.w, f, r.w);
        }
        if (outer > 1) {
            float* part = a.parts + (((size_t)row * a.nh + head0 + h) * outer + split / cluster) * (HD + 2);
            if (c == 0) { part[0] = most; part[1] = sum; }
            part[2 + c] = r.x; part[3 + c] = r.y; part[4 + c] = r.z; part[5 + c] = r.w;
        } else {
            const float inv = sum != 0.f ? 1.0f / sum : 0.f;
            __nv_bfloat16* out = (__nv_bfloat16*)a.out + (size_t)row * a.out_stride + (size_t)(head0 + h) * HD + c;
            const uint32_t lo = kv4_pack(r.x * inv, r.y * inv), hi = kv4_pack(r.z * inv, r.w * inv);
            if ((((uintptr_t)a.out | (uintptr_t)(a.out_stride * 2)) & 7) == 0) {
                *reinterpret_cast<uint2*>(out) = make_uint2(lo, hi);
            } else {
                unsigned short* s = reinterpret_cast<unsigned short*>(out);
                s[0] = (unsigned short)lo; s[1] = (unsigned short)(lo >> 16); s[2] = (unsigned short)hi; s[3] = (unsigned short)(hi >> 16);
            }
        }
    }
    if (cluster > 1) asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");   // (its memory is read until here)
}

template <int HD>
static int kv4_decode_launch(const Kv4AttnArgs& a, int splits, int cluster, cudaStream_t stream) {
    using Geo = Kv4Geometry<HD>;
    static_assert(Geo::RING % 128 == 0 && Geo::TILE % 16 == 0, "tiles start where bulk copies may");
    const cudaError_t e = cudaFuncSetAttribute(kv4_decode_mma_kernel<HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, Geo::SMEM);
    GB_REQUIRE(e == cudaSuccess, "gb_kv4_attention_decode: %d bytes of shared memory refused: %s", Geo::SMEM, cudaGetErrorString(e));
    const int group = a.nh / a.nkv;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(splits, a.nkv * ((group + KV4M_HEADS - 1) / KV4M_HEADS), a.n);
    cfg.blockDim = dim3(KV4M_WARPS * 32);
    cfg.dynamicSmemBytes = Geo::SMEM;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    int na = 0;
    if (gb_pdl_enabled() & GB_PDL_ATTENTION) {
        attr[na].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[na].val.programmaticStreamSerializationAllowed = 1;
        ++na;
    }
    if (cluster > 1) {
        attr[na].id = cudaLaunchAttributeClusterDimension;
        attr[na].val.clusterDim.x = cluster;
        attr[na].val.clusterDim.y = attr[na].val.clusterDim.z = 1;
        ++na;
    }
    cfg.attrs = attr;
    cfg.numAttrs = na;
    const cudaError_t rc = cudaLaunchKernelEx(&cfg, kv4_decode_mma_kernel<HD>, a, cluster);
    if (rc != cudaSuccess) {
        gb_set_error("gb_kv4_attention_decode: launch failed: %s", cudaGetErrorString(rc));
        return 2;
    }
    if (int bad = gb_check_launch("gb_kv4_attention_decode")) return bad;
    return splits > cluster ? kv4_merge(a, GB_BF16, splits / cluster, stream) : 0;
}

// As gb_kv4_attention_rows, q and out bfloat16, the keys of a row in `splits` shares that are added up in clusters of `cluster` blocks (1, 2, 4 or 8; a
// divisor of splits). parts (splits > cluster): float32 [n, nh, splits / cluster, hd + 2].
GB_EXPORT int gb_kv4_attention_decode(const void* q, long long q_stride, void* out, long long out_stride, const void* kcache, const void* vcache,
                                      const int* block_tables, int max_pages, const int* row_seq, const int* positions, int n, int nh, int nkv,
                                      int hd, int page_size, long long num_pages, float scale, int window, int splits, int cluster, float* parts,
                                      int* status, cudaStream_t stream) {
    KV4_REQUIRE_SIZES("gb_kv4_attention_decode")
    GB_REQUIRE(n >= 0 && nh > 0 && nh % nkv == 0 && max_pages > 0, "gb_kv4_attention_decode: bad sizes (rows %d, heads %d of %d, tables of %d pages)", n, nh, nkv, max_pages);
    GB_REQUIRE((cluster == 1 || cluster == 2 || cluster == 4 || cluster == 8) && splits >= cluster && splits % cluster == 0,
               "gb_kv4_attention_decode: %d shares in clusters of %d are not built", splits, cluster);
    GB_REQUIRE(splits == cluster || parts != nullptr, "gb_kv4_attention_decode: %d shares need their scratch", splits);
    GB_REQUIRE((long long)max_pages * page_size < (1ll << 31) - 64, "gb_kv4_attention_decode: block tables of %d pages reach too far", max_pages);
    GB_REQUIRE(n <= 65535 && nh <= 65535, "gb_kv4_attention_decode: %d rows of %d heads are too many for one launch", n, nh);
    GB_REQUIRE(((uintptr_t)kcache | (uintptr_t)vcache) % 16 == 0, "gb_kv4_attention_decode: the cache must be 16-byte aligned");
    if (n == 0) return 0;
    Kv4AttnArgs a = {};
    a.q = q; a.q_stride = q_stride; a.out = out; a.out_stride = out_stride; a.kcache = (const unsigned char*)kcache;
    a.vcache = (const unsigned char*)vcache; a.block_tables = block_tables; a.max_pages = max_pages; a.row_seq = row_seq; a.positions = positions;
    a.n = n; a.nh = nh; a.nkv = nkv; a.hd = hd; a.page_size = page_size; a.num_pages = num_pages; a.scale = scale * KV4_LOG2E;
    a.window = window > 0 ? window : 0; a.parts = parts; a.status = status;
    if (hd == 32) return kv4_decode_launch<32>(a, splits, cluster, stream);
    if (hd == 64) return kv4_decode_launch<64>(a, splits, cluster, stream);
    if (hd == 96) return kv4_decode_launch<96>(a, splits, cluster, stream);
    if (hd == 128) return kv4_decode_launch<128>(a, splits, cluster, stream);
    if (hd == 256) return kv4_decode_launch<256>(a, splits, cluster, stream);
    GB_REQUIRE(false, "gb_kv4_attention_decode: head size %d is not built (32, 64, 96, 128, 256)", hd);
}
