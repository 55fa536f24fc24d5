// Decode attention over a cache in 4 bits (layout: kv4.cuh) in bfloat16 on the tensor cores.
//
// One block = one row, up to eight query heads of one kv head, one share of the row's keys; its warps take the share's steps of 32 keys (16 of
// the larger head sizes) in turn. A tile of 16 keys is one contiguous piece of the pool, as are its values, and each warp has a ring of STAGES steps in shared memory
// that its lanes keep full with asynchronous copies of 16 bytes: one multiplication an address, and what a multiprocessor has in
// flight (16 warps x 2 or 3 steps x 36 hd bytes) is several times what the memory's latency asks for.
//
// Codes become operands of mma.sync m16n8k16 without being scaled: a code u in four bits, put under 0x4300, is the bfloat16 128 + u.
//   * S^T = K Q^T, 16 keys as the rows, the heads as columns: the sums of a group of 32 channels start at -136 sum q and add q (128 + u)
//     (u = s + 8; float32 sums of exact products, so this costs 5 of their 24 bits), and the key's scale is applied to what comes out:
//     one multiplication a key, head and group instead of one a number.
//   * O^T = V^T P^T, 16 channels of a group as the rows, the heads as columns: p times the value's scale is rounded to bfloat16 (the
//     only rounding of the kernel besides the result's: half a step is 2^-9 of the weight, as in every kernel here that multiplies weights on
//     the tensor cores) and turned over in registers, codes less 136 are whole numbers that bfloat16 holds. (Values cannot keep their 128 + 8: the
//     sum over thousands of keys would be 136 sum p against results near zero.)
// (With the queries as the 16 rows of A, eight of them zero, the scores lie as the second product wants them, but take twice the products, twice
// the scales and a move for each operand register: 64 rows of 32/32 heads of 64, 4,096 keys in even shares 182 to 200 us.)
// The reference that is subtracted from scores rises only when one exceeds it by 2^8 (weights up to 256 cost the float32 sums nothing), so that
// the sums of O are hardly ever rescaled.
// The warps of a block add up in shared memory. How the keys are shared among blocks: a cluster of up to eight blocks a row and chunk of heads, which
// add up from each other's shared memory, or, behind the longest contexts, all rows' steps cut evenly among the blocks that run at once
// (kv4_decode_even_kernel). Nothing is left behind for the next call.
//
// What bounds it: instructions, some 430 for 32 keys of a head of 64 and their values, and how they wait for one another: 2.4 of 4 are issued a cycle
// and multiprocessor (all 4 would be 97 of the 154 us below, the memory's share is 92). 64 rows of 32/32 heads of 64 behind 4,096 keys, 605 MB, take 154 us (3.9 TB/s); 2 rows of 32/8 heads of 128 behind 131,072, 302 MB, 86 us
// (157 and 87 with one float32 where two go into an instruction, which is the form that the next figures are from).
// The second without taking codes apart 72, without the second product 63, without copies 80; one multiprocessor's blocks 3 / 4 / 5 of them 91 / 87 /
// 115, of heads of 64 (the first) 4 / 5 / 6 159 / 157 / 165; a ring of five steps 163; in even shares with one tile a step instead of two 180 to 203.
#include <atomic>

#include "kv4_attention.cuh"

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

constexpr int KV4M_WARPS = 4;
constexpr int KV4M_HEADS = 8;      // query heads of a block

__device__ __forceinline__ void kv4_mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void kv4_mma_from(float (&d)[4], const float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};\n"
                 : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
}
__device__ __forceinline__ void kv4_copy16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
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

// An 8 x 8 matrix of bfloat16, two neighbours of a row a lane, turned over.
__device__ __forceinline__ uint32_t kv4_turned(uint32_t v) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}

template <int W> __device__ __forceinline__ void kv4_words(const unsigned char* p, uint32_t (&w)[W]);
// G scales of one token (2 G bytes, aligned to that where G is even)
template <int G> __device__ __forceinline__ void kv4_scales(const unsigned char* p, float (&d)[G]) {
    if constexpr (G % 2 == 0) {
        uint32_t w[G / 2];
        kv4_words<G / 2>(p, w);
#pragma unroll
        for (int i = 0; i < G; ++i) d[i] = kv4_bf16(w, i);
    } else {
#pragma unroll
        for (int i = 0; i < G; ++i) d[i] = __uint_as_float((uint32_t)reinterpret_cast<const unsigned short*>(p)[i] << 16);
    }
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
    static constexpr int TILES = HD <= 64 ? 2 : 1;                        // of a warp's step (two of the larger ones would not fit its registers)
    static constexpr int KEYS = TILES * KV4_TILE;
    static constexpr int STEP = TILES * 2 * TILE;                         // bytes of a step's keys and values
    static constexpr int STAGES = HD <= 128 ? 4 : 3;
    static constexpr int RING = STAGES * STEP;                            // of a warp
    static constexpr int PART = KV4M_HEADS * (HD + 2) * 4;                // bytes of a warp's, or the block's, result: maxima, sums, rows
    static constexpr int BLOCKS = HD <= 32 ? 6 : HD <= 96 ? 5 : HD <= 128 ? 4 : 2;     // of a multiprocessor
    static constexpr int SMEM = KV4M_WARPS * RING > (KV4M_WARPS + 1) * PART ? KV4M_WARPS * RING : (KV4M_WARPS + 1) * PART;
};

// The keys that a row sees, in steps of KEYS of them: the first key, the first step, and how many. A position that the block table does not reach is
// reported and the row reads nothing, as a padding row.
struct Kv4Row { int pos, first, step0, steps; };
template <int KEYS>
__device__ __forceinline__ Kv4Row kv4_row(const Kv4AttnArgs& a, int row, bool tell) {
    Kv4Row r;
    r.pos = a.positions[row];
    if (r.pos >= 0 && r.pos / a.page_size >= a.max_pages) {
        if (tell) atomicOr(a.status, GB_STATUS_BAD_POSITION);
        r.pos = -1;
    }
    r.first = gb_first_key(r.pos, a.window);
    r.step0 = r.first / KEYS;
    r.steps = r.pos < 0 ? 0 : r.pos / KEYS - r.step0 + 1;
    return r;
}

// One block: steps begin .. end - 1 of a row for `heads` query heads of kv head kvh, the first of them head0. Leaves maxima [8], sums [8] and rows
// [8][HD] not yet divided in shared memory, where it returns; what the block wrote there before must have been read.
template <int HD>
__device__ __forceinline__ float* kv4_segment(const Kv4AttnArgs& a, unsigned char* smem, const int row, const int kvh, const int head0, const int heads,
                                              const int pos, const int first, const int begin, const int end) {
    using Geo = Kv4Geometry<HD>;
    constexpr int G = Geo::G, STAGES = Geo::STAGES, TILE = Geo::TILE, KEYS = Geo::KEYS, TILES = Geo::TILES, BATCH = 32 / TILES;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int mine = end - begin > warp ? (end - begin - warp + KV4M_WARPS - 1) / KV4M_WARPS : 0;      // steps begin + warp + KV4M_WARPS * i
    const int* table = a.block_tables + (size_t)(pos < 0 ? 0 : a.row_seq[row]) * a.max_pages;
    const int per_page = a.page_size / KV4_TILE;

    // Where the tiles of this warp's steps lie, a batch of 32 tiles at a time: lane TILES * i + j has tile j of step i, as its number in the pool,
    // or -1 where it holds no key in sight or its page is missing.
    auto look = [&](int i) -> int {
        const int tile = TILES * (begin + warp + KV4M_WARPS * (i + lane / TILES)) + lane % TILES;
        if (i + lane / TILES >= mine || tile * KV4_TILE > pos || (tile + 1) * KV4_TILE <= first) return -1;
        const int pi = tile / per_page;
        const long long page = table[pi];
        if (page < 0 || page >= a.num_pages) {
            atomicOr(a.status, GB_STATUS_BAD_SLOT);
            return -1;
        }
        return (int)((page * a.nkv + kvh) * per_page + (tile - pi * per_page));
    };
    int place = look(0), place_next = look(BATCH);
    unsigned lack = __ballot_sync(0xffffffffu, place < 0), lack_ahead = lack;      // of the batch that is worked on, that is asked for
    // A tile's keys and values, 16 bytes a lane and turn, one turn of which may bring the end of the one and the start of the other.
    constexpr int PIECES = TILE / 16, TURNS = (2 * PIECES + 31) / 32, MIXED = PIECES % 32 ? PIECES / 32 : -1;
    const unsigned char* const keys = a.kcache + lane * 16;
    const unsigned char* const values = a.vcache + lane * 16 - TILE;
    const uint32_t ring = smem_u32(smem + warp * Geo::RING) + lane * 16;
    auto ask = [&](int i, int stage) {       // (all lanes)
        const uint32_t dst = ring + stage * Geo::STEP;
#pragma unroll
        for (int j = 0; j < TILES; ++j) {
            const int at = __shfl_sync(0xffffffffu, place, TILES * (i & (BATCH - 1)) + j);
            if (at >= 0) {
                const unsigned char* k = keys + (unsigned long long)(unsigned)at * TILE;
                const unsigned char* v = values + (unsigned long long)(unsigned)at * TILE;
#pragma unroll
                for (int c = 0; c < TURNS; ++c) {
                    const unsigned char* from = c == MIXED ? (lane + 32 * c < PIECES ? k : v) : c < PIECES / 32 ? k : v;
                    if (c + 1 < TURNS || 2 * PIECES % 32 == 0 || lane + 32 * c < 2 * PIECES) kv4_copy16(dst + j * 2 * TILE + c * 512, from + c * 512);
                }
            }
        }
    };
#pragma unroll
    for (int i = 0; i < STAGES - 1; ++i) {
        if (i < mine) ask(i, i);
        asm volatile("cp.async.commit_group;" ::: "memory");
    }

    // Q^T as the B operand: column g is head head0 + g; the two k16 steps of a group take channels 8 t + {0, 4, 1, 5} and {2, 6, 3, 7} of it
    // at this thread's places, as a word of eight codes yields them.
    uint32_t qf[G][4];
    float from[G][4];                        // -136 times a group's sum of q, heads 2 t and 2 t + 1: where the sums of its products start
    const float scale = a.scale;
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
            from[i][0] = from[i][2] = -136.f * __shfl_sync(0xffffffffu, sum, 8 * t);
            from[i][1] = from[i][3] = -136.f * __shfl_sync(0xffffffffu, sum, 8 * t + 4);
        }
    }

    float m[2] = {KV4_NEG_BIG, KV4_NEG_BIG}, l[2] = {0.f, 0.f};      // of heads 2 t and 2 t + 1; l: this thread's keys
    float o[G][2][4];                        // [group][pair of channels]: channel 32 i + 4 g + 2 j (and + 1 in [2], [3]) of heads 2 t, 2 t + 1
#pragma unroll
    for (int i = 0; i < G; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[i][j][e] = 0.f;

    int stage = 0, stage_ahead = STAGES - 1;
    const unsigned char* const kbase = smem + warp * Geo::RING + g * (HD / 2) + t * G * 4;           // this thread's codes of key g
    const unsigned char* const vbase = smem + warp * Geo::RING + TILE + 2 * t * (HD / 2) + g * G * 2;   // ... of value 2 t
    const unsigned char* const dbase = smem + warp * Geo::RING + 8 * HD + g * G * 2;               // scales of key g
    for (int i = 0; i < mine; ++i) {
        const int ahead = i + STAGES - 1;
        if (ahead < mine) {                  // into the stage that was read an iteration ago, by all lanes: the barrier at the end of it
            if ((ahead & (BATCH - 1)) == 0) {      // (the next batch's places, while this one is worked on)
                place = place_next;
                place_next = look(ahead + BATCH);
                lack_ahead = __ballot_sync(0xffffffffu, place < 0);
            }
            ask(ahead, stage_ahead);
        }
        if ((i & (BATCH - 1)) == 0) lack = lack_ahead;
        asm volatile("cp.async.commit_group;\n\tcp.async.wait_group %0;" ::"n"(STAGES - 1) : "memory");
        __syncwarp();                        // what every lane has brought is there for all
        const int offset = stage * Geo::STEP;
        const int key0 = (begin + warp + KV4M_WARPS * i) * KEYS;
        const unsigned have = ~(lack >> (TILES * (i & (BATCH - 1)))) & ((1u << TILES) - 1);
        // At an end of what is in sight, or where a page is missing: the scale of a value that is not in sight may be anything, and becomes zero
        // (its weight is zero); scores are masked below. Both are branches hardly ever taken.
        const bool edge = key0 < first || key0 + KEYS - 1 > pos || have != (1u << TILES) - 1;
        if (edge) {
            if (lane < KEYS) {
                const int key = key0 + lane;
                if (key < first || key > pos || !(have >> (lane / KV4_TILE) & 1u)) {
                    unsigned short* d = reinterpret_cast<unsigned short*>(smem + warp * Geo::RING + offset + lane / KV4_TILE * 2 * TILE + TILE + 8 * HD) + lane % KV4_TILE * G;
#pragma unroll
                    for (int k = 0; k < G; ++k) d[k] = 0;
                }
            }
            __syncwarp();
        }
        // ---- scores of keys g and g + 8 of tile x, heads 2 t and 2 t + 1
        float2 sc[TILES][2];
#pragma unroll
        for (int x = 0; x < TILES; ++x) {
            uint32_t w[2][G];
            float d[2][G];
#pragma unroll
            for (int y = 0; y < 2; ++y) {
                kv4_words<G>(kbase + offset + x * 2 * TILE + y * 8 * (HD / 2), w[y]);
                kv4_scales<G>(dbase + offset + x * 2 * TILE + y * 8 * G * 2, d[y]);
            }
#pragma unroll
            for (int k = 0; k < G; ++k) {
                float c[4];
                kv4_mma_from(c, from[k], kv4_up(w[0][k], 0), kv4_up(w[1][k], 0), kv4_up(w[0][k], 1), kv4_up(w[1][k], 1), qf[k][0], qf[k][1]);
                kv4_mma(c, kv4_up(w[0][k], 2), kv4_up(w[1][k], 2), kv4_up(w[0][k], 3), kv4_up(w[1][k], 3), qf[k][2], qf[k][3]);
#pragma unroll
                for (int y = 0; y < 2; ++y) {
                    const float2 both = make_float2(d[y][k], d[y][k]), of = make_float2(c[2 * y], c[2 * y + 1]);
                    sc[x][y] = k == 0 ? __fmul2_rn(both, of) : __ffma2_rn(both, of, sc[x][y]);
                }
            }
        }
        if (edge) {
            asm volatile("" ::: "memory");   // (a branch, not selections in every step)
#pragma unroll
            for (int x = 0; x < TILES; ++x)
#pragma unroll
                for (int y = 0; y < 2; ++y) {
                    const int key = key0 + KV4_TILE * x + 8 * y + g;
                    if (key < first || key > pos || !(have >> x & 1u)) sc[x][y] = make_float2(-INFINITY, -INFINITY);
                }
        }
        // ---- weights
        float most[2] = {fmaxf(sc[0][0].x, sc[0][1].x), fmaxf(sc[0][0].y, sc[0][1].y)};
#pragma unroll
        for (int x = 1; x < TILES; ++x) {
            most[0] = fmaxf(most[0], fmaxf(sc[x][0].x, sc[x][1].x));
            most[1] = fmaxf(most[1], fmaxf(sc[x][0].y, sc[x][1].y));
        }
        if (__any_sync(0xffffffffu, fmaf(most[0], scale, -m[0]) > 8.f || fmaf(most[1], scale, -m[1]) > 8.f)) {
            float corr[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                float v = most[e] * scale;
#pragma unroll
                for (int x = 4; x < 32; x <<= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, x));
                v = fmaxf(m[e], v);
                corr[e] = kv4_exp2(m[e] - v);
                m[e] = v;
                l[e] *= corr[e];
            }
#pragma unroll
            for (int k = 0; k < G; ++k)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    o[k][j][0] *= corr[0]; o[k][j][1] *= corr[1]; o[k][j][2] *= corr[0]; o[k][j][3] *= corr[1];
                }
        }
        // ---- output: weights times the values' scales as the B operand, codes of keys 2 t, 2 t + 1, 2 t + 8, 2 t + 9 as the A operand
#pragma unroll
        for (int x = 0; x < TILES; ++x) {
            uint32_t b[2][G];
#pragma unroll
            for (int y = 0; y < 2; ++y) {
                float d[G];
                const float2 over = __ffma2_rn(sc[x][y], make_float2(scale, scale), make_float2(-m[0], -m[1]));
                const float2 p = make_float2(kv4_exp2(over.x), kv4_exp2(over.y)), sum = __fadd2_rn(make_float2(l[0], l[1]), p);
                l[0] = sum.x;
                l[1] = sum.y;
                kv4_scales<G>(dbase + offset + TILE + x * 2 * TILE + y * 8 * G * 2, d);
#pragma unroll
                for (int k = 0; k < G; ++k) {
                    const float2 w = __fmul2_rn(p, make_float2(d[k], d[k]));
                    b[y][k] = kv4_turned(kv4_pack(w.x, w.y));
                }
            }
            const unsigned char* vr = vbase + offset + x * 2 * TILE;
            uint32_t w[4][(G + 1) / 2];      // half words of the four keys, two groups a word
            if constexpr (G % 2 == 0) {
                kv4_words<G / 2>(vr, w[0]);
                kv4_words<G / 2>(vr + HD / 2, w[1]);
                kv4_words<G / 2>(vr + 8 * (HD / 2), w[2]);
                kv4_words<G / 2>(vr + 9 * (HD / 2), w[3]);
            } else {
#pragma unroll
                for (int y = 0; y < 4; ++y) {
                    const unsigned short* h = reinterpret_cast<const unsigned short*>(vr + ((y & 1) + 8 * (y >> 1)) * (HD / 2));
#pragma unroll
                    for (int k = 0; k < (G + 1) / 2; ++k) w[y][k] = h[2 * k] | (2 * k + 1 < G ? (uint32_t)h[2 * k + 1] << 16 : 0u);
                }
            }
#pragma unroll
            for (int k = 0; k < G; ++k) {
                const uint32_t lo = __byte_perm(w[0][k / 2], w[1][k / 2], k & 1 ? 0x7632 : 0x5410);
                const uint32_t hi = __byte_perm(w[2][k / 2], w[3][k / 2], k & 1 ? 0x7632 : 0x5410);
#pragma unroll
                for (int j = 0; j < 2; ++j)
                    kv4_mma(o[k][j], kv4_down(kv4_up(lo, 2 * j)), kv4_down(kv4_up(lo, 2 * j + 1)), kv4_down(kv4_up(hi, 2 * j)),
                            kv4_down(kv4_up(hi, 2 * j + 1)), b[0][k], b[1][k]);
            }
        }
        __syncwarp();                        // every lane has read this stage
        stage_ahead = stage;
        if (++stage == STAGES) stage = 0;
    }
    // ---- the warps' results: maxima [8], sums [8], rows [8][HD] each
#pragma unroll
    for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) l[e] += __shfl_xor_sync(0xffffffffu, l[e], x);
    __syncthreads();
    float* parts = reinterpret_cast<float*>(smem);
    constexpr int PART = Geo::PART / 4;
    {
        float* w = parts + warp * PART;
        if (g == 0) {
            *reinterpret_cast<float2*>(w + 2 * t) = make_float2(m[0], m[1]);
            *reinterpret_cast<float2*>(w + 8 + 2 * t) = make_float2(l[0], l[1]);
        }
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
    __syncthreads();
    return block;
}

// Four numbers of a head's row from channel c on, divided by the sum, to their place.
__device__ __forceinline__ void kv4_out(const Kv4AttnArgs& a, int row, int head, int c, const float4& r, float sum) {
    const float inv = sum != 0.f ? 1.0f / sum : 0.f;
    __nv_bfloat16* out = (__nv_bfloat16*)a.out + (size_t)row * a.out_stride + (size_t)head * a.hd + c;
    const uint32_t lo = kv4_pack(r.x * inv, r.y * inv), hi = kv4_pack(r.z * inv, r.w * inv);
    if ((((uintptr_t)a.out | (uintptr_t)(a.out_stride * 2)) & 7) == 0) {
        *reinterpret_cast<uint2*>(out) = make_uint2(lo, hi);
    } else {
        unsigned short* s = reinterpret_cast<unsigned short*>(out);
        s[0] = (unsigned short)lo; s[1] = (unsigned short)(lo >> 16); s[2] = (unsigned short)hi; s[3] = (unsigned short)(hi >> 16);
    }
}

// A cluster of blocks (or one) for each row and up to eight heads of a kv head, the row's steps in equal shares.
template <int HD>
__global__ void __launch_bounds__(KV4M_WARPS * 32, Kv4Geometry<HD>::BLOCKS) kv4_decode_cluster_kernel(const Kv4AttnArgs a) {
    extern __shared__ __align__(128) unsigned char smem[];
    gb_pdl_wait();
    gb_pdl_launch_dependents();
    const int group = a.nh / a.nkv, chunks = (group + KV4M_HEADS - 1) / KV4M_HEADS;
    const int kvh = blockIdx.y / chunks, head0 = kvh * group + (blockIdx.y % chunks) * KV4M_HEADS;
    const int heads = min(KV4M_HEADS, (kvh + 1) * group - head0), row = blockIdx.z, rank = blockIdx.x, cluster = gridDim.x;
    const Kv4Row r = kv4_row<Kv4Geometry<HD>::KEYS>(a, row, threadIdx.x == 0 && blockIdx.x == 0 && blockIdx.y == 0);
    float* block = kv4_segment<HD>(a, smem, row, kvh, head0, heads, r.pos, r.first, r.step0 + kv4_share(r.steps, rank, cluster),
                                   r.step0 + kv4_share(r.steps, rank + 1, cluster));
    // each block adds up every cluster-th piece from all of them, in their order
    if (cluster > 1) asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
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
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int w = 0; w < cluster; ++w) most = fmaxf(most, get(w, h));
        for (int w = 0; w < cluster; ++w) {
            const float f = kv4_exp2(get(w, h) - most);
            const float4 v = get4(w, 16 + h * HD + c);
            sum = fmaf(get(w, 8 + h), f, sum);
            o.x = fmaf(v.x, f, o.x); o.y = fmaf(v.y, f, o.y); o.z = fmaf(v.z, f, o.z); o.w = fmaf(v.w, f, o.w);
        }
        kv4_out(a, row, head0 + h, c, o, sum);
    }
    if (cluster > 1) asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");   // (its memory is read until here)
}

// Even shares of all rows' steps. The steps of all rows, kv heads and chunks of eight heads, one after the other, are cut into as many
// equal pieces as there are blocks, whatever the rows' lengths: block b takes steps b S / B to (b + 1) S / B - 1 of the S. What a block has of a (row,
// chunk) that it does not have as a whole it leaves in `parts` (a result of a segment that starts its piece in its first place, else in its
// second), and the block that has the beginning writes down what kv4_even_merge_kernel is to add up.
constexpr int KV4E_ROWS = 1024;     // rows at most (their sums of steps lie in shared memory)

// sums[r]: steps of rows 0 .. r - 1, r = 0 .. n; a row without keys counts as one step, which writes its zeros.
template <int KEYS>
__device__ __forceinline__ void kv4_sums(const Kv4AttnArgs& a, int* sums, bool tell) {
    __shared__ int warps[KV4M_WARPS];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, each = (a.n + KV4M_WARPS * 32 - 1) / (KV4M_WARPS * 32);
    int mine = 0;
    for (int i = tid * each; i < min(a.n, (tid + 1) * each); ++i) {
        mine += max(1, kv4_row<KEYS>(a, i, tell).steps);
        sums[i + 1] = mine;
    }
    int up = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, up, o);
        if (lane >= o) up += v;
    }
    if (lane == 31) warps[warp] = up;
    if (tid == 0) sums[0] = 0;
    __syncthreads();
    int before = up - mine;
    for (int w = 0; w < warp; ++w) before += warps[w];
    for (int i = tid * each; i < min(a.n, (tid + 1) * each); ++i) sums[i + 1] += before;
    __syncthreads();
}
__device__ __forceinline__ int kv4_row_of(const int* sums, int n, long long flat, int per) {      // the row of step `flat`, `per` chunks a row
    int lo = 0, hi = n - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        if ((long long)sums[mid] * per <= flat) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}
// floats of a place in `parts`
template <int HD> constexpr int KV4E_PART = KV4M_HEADS * (HD + 2);

template <int HD>
__global__ void __launch_bounds__(KV4M_WARPS * 32, Kv4Geometry<HD>::BLOCKS) kv4_decode_even_kernel(const Kv4AttnArgs a) {
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ int sums[KV4E_ROWS + 1];
    gb_pdl_wait();
    gb_pdl_launch_dependents();
    const int group = a.nh / a.nkv, chunks = (group + KV4M_HEADS - 1) / KV4M_HEADS, per = a.nkv * chunks;
    kv4_sums<Kv4Geometry<HD>::KEYS>(a, sums, blockIdx.x == 0);
    const long long all = (long long)sums[a.n] * per;
    const int blocks = (int)min((long long)gridDim.x, all);
    int4* jobs = reinterpret_cast<int4*>(a.parts + 2ll * gridDim.x * KV4E_PART<HD>);
    volatile __shared__ long long where;     // the step that is next: not worth a register while keys are walked through
    if (threadIdx.x == 0) {
        where = all * blockIdx.x / blocks;
        jobs[blockIdx.x] = make_int4(-1, 0, 0, 0);
    }
    __syncthreads();
    while (blockIdx.x < blocks) {
        const long long at = where, from = all * blockIdx.x / blocks, to = all * (blockIdx.x + 1) / blocks;
        if (at >= to) break;
        const int row = kv4_row_of(sums, a.n, at, per), size = sums[row + 1] - sums[row];
        const long long rest = at - (long long)sums[row] * per;
        const int y = (int)(rest / size), step = (int)(rest - (long long)y * size);
        const int count = (int)min((long long)(size - step), to - at);
        const bool first_piece = at == from, whole = count == size;
        const int kvh = y / chunks, head0 = kvh * group + (y % chunks) * KV4M_HEADS, heads = min(KV4M_HEADS, (kvh + 1) * group - head0);
        __syncthreads();                     // (all have read where)
        if (threadIdx.x == 0) {
            where = at + count;
            if (step == 0 && !whole)         // the block that holds the last step is the last one that begins at or before it
                jobs[blockIdx.x] = make_int4(row, head0 * 16 + heads, first_piece ? 0 : 1, (int)(((at + size) * blocks - 1) / all));
        }
        const Kv4Row r = kv4_row<Kv4Geometry<HD>::KEYS>(a, row, false);
        const float* block = kv4_segment<HD>(a, smem, row, kvh, head0, heads, r.pos, r.first, r.step0 + step, r.step0 + (r.steps > 0 ? step + count : 0));
        float* part = a.parts + (2ll * blockIdx.x + (first_piece ? 0 : 1)) * KV4E_PART<HD>;
        for (int i = threadIdx.x; i < heads * (HD / 4); i += KV4M_WARPS * 32) {
            const int h = i / (HD / 4), c = i % (HD / 4) * 4;
            const float4 o = *reinterpret_cast<const float4*>(block + 16 + h * HD + c);
            if (whole) {
                kv4_out(a, row, head0 + h, c, o, block[8 + h]);
            } else {
                *reinterpret_cast<float4*>(part + 16 + h * HD + c) = o;
                if (c == 0) { part[h] = block[h]; part[8 + h] = block[8 + h]; }
            }
        }
        __syncthreads();
    }
}

// Block (b, h) adds up head h of the pieces of what block b of the kernel above begins and others go on with: 16 groups of threads (of HD / 4, four
// channels each) take the pieces in turn, then one adds up the groups. The first piece may be in its block's second place, all others
// start their blocks.
constexpr int KV4E_GROUPS = 16;
template <int HD>
__global__ void __launch_bounds__(KV4E_GROUPS * HD / 4) kv4_even_merge_kernel(const Kv4AttnArgs a) {
    __shared__ float ml[KV4E_GROUPS][2];
    __shared__ float4 rows[KV4E_GROUPS][HD / 4];
    gb_pdl_launch_dependents();
    gb_pdl_wait();
    const int4 job = reinterpret_cast<const int4*>(a.parts + 2ll * gridDim.x * KV4E_PART<HD>)[blockIdx.x];
    const int h = blockIdx.y, b0 = blockIdx.x, pieces = job.w - b0 + 1;
    if (job.x < 0 || h >= job.y % 16) return;
    const int group = threadIdx.x / (HD / 4), c = threadIdx.x % (HD / 4);
    auto piece = [&](int i) { return a.parts + (2ll * (b0 + i) + (i == 0 ? job.z : 0)) * KV4E_PART<HD>; };
    float most = KV4_NEG_BIG, sum = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    constexpr int FLY = 4;                   // pieces under way at once
    for (int i0 = group; i0 < pieces; i0 += FLY * KV4E_GROUPS) {
        float m[FLY], l[FLY];
        float4 v[FLY];
#pragma unroll
        for (int u = 0; u < FLY; ++u) {
            const int i = i0 + u * KV4E_GROUPS;
            m[u] = KV4_NEG_BIG; l[u] = 0.f; v[u] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (i < pieces) {
                const float* p = piece(i);
                m[u] = p[h]; l[u] = p[8 + h];
                v[u] = *reinterpret_cast<const float4*>(p + 16 + h * HD + 4 * c);
            }
        }
        float up = most;
#pragma unroll
        for (int u = 0; u < FLY; ++u) up = fmaxf(up, m[u]);
        const float f0 = kv4_exp2(most - up);
        most = up;
        sum *= f0; o.x *= f0; o.y *= f0; o.z *= f0; o.w *= f0;
#pragma unroll
        for (int u = 0; u < FLY; ++u) {
            const float f = kv4_exp2(m[u] - up);
            sum = fmaf(l[u], f, sum);
            o.x = fmaf(v[u].x, f, o.x); o.y = fmaf(v[u].y, f, o.y); o.z = fmaf(v[u].z, f, o.z); o.w = fmaf(v[u].w, f, o.w);
        }
    }
    if (c == 0) { ml[group][0] = most; ml[group][1] = sum; }
    rows[group][c] = o;
    __syncthreads();
    if (group > 0) return;
    const int used = min(pieces, KV4E_GROUPS);
    for (int g = 1; g < used; ++g) most = fmaxf(most, ml[g][0]);
    sum = 0.f;
    o = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int g = 0; g < used; ++g) {
        const float f = kv4_exp2(ml[g][0] - most);
        const float4 v = rows[g][c];
        sum = fmaf(ml[g][1], f, sum);
        o.x = fmaf(v.x, f, o.x); o.y = fmaf(v.y, f, o.y); o.z = fmaf(v.z, f, o.z); o.w = fmaf(v.w, f, o.w);
    }
    kv4_out(a, job.x, job.y / 16 + h, 4 * c, o, sum);
}

// Blocks of a kernel that run at once, asked once a head size.
template <int HD>
static int kv4_resident() {
    static std::atomic<int> known{0};
    int n = known.load(std::memory_order_relaxed);
    if (n == 0) {
        int device = 0, sms = 0, each = 0;
        if (cudaGetDevice(&device) != cudaSuccess || cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device) != cudaSuccess ||
            cudaFuncSetAttribute(kv4_decode_even_kernel<HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, Kv4Geometry<HD>::SMEM) != cudaSuccess ||
            cudaOccupancyMaxActiveBlocksPerMultiprocessor(&each, kv4_decode_even_kernel<HD>, KV4M_WARPS * 32, Kv4Geometry<HD>::SMEM) != cudaSuccess) {
            cudaGetLastError();
            return 0;
        }
        n = sms * each;
        known.store(n, std::memory_order_relaxed);
    }
    return n;
}

// How many blocks share the steps of n rows evenly where no row has more than `reach` keys in sight: what runs at once, none with fewer than
// 8 steps (two a warp) of full rows.
template <int HD>
static int kv4_even_blocks(int n, int nh, int nkv, long long reach) {
    const long long chunks = (nh / nkv + KV4M_HEADS - 1) / KV4M_HEADS, steps = (reach + Kv4Geometry<HD>::KEYS - 1) / Kv4Geometry<HD>::KEYS * n * nkv * chunks;
    const long long most = steps / 8 > 1 ? steps / 8 : 1, at_once = kv4_resident<HD>();
    return (int)(at_once < most ? at_once : most);
}

template <int HD>
static int kv4_decode_launch(const Kv4AttnArgs& a, int cluster, int blocks, cudaStream_t stream) {
    using Geo = Kv4Geometry<HD>;
    static_assert(Geo::RING % 128 == 0 && Geo::TILE % 16 == 0, "tiles start where copies may");
    void (*kernel)(const Kv4AttnArgs) = blocks ? kv4_decode_even_kernel<HD> : kv4_decode_cluster_kernel<HD>;
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Geo::SMEM);
    GB_REQUIRE(e == cudaSuccess, "gb_kv4_attention_decode: %d bytes of shared memory refused: %s", Geo::SMEM, cudaGetErrorString(e));
    const int group = a.nh / a.nkv;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = blocks ? dim3(blocks) : dim3(cluster, a.nkv * ((group + KV4M_HEADS - 1) / KV4M_HEADS), a.n);
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
    if (!blocks && cluster > 1) {
        attr[na].id = cudaLaunchAttributeClusterDimension;
        attr[na].val.clusterDim.x = cluster;
        attr[na].val.clusterDim.y = attr[na].val.clusterDim.z = 1;
        ++na;
    }
    cfg.attrs = attr;
    cfg.numAttrs = na;
    const cudaError_t rc = cudaLaunchKernelEx(&cfg, kernel, a);
    if (rc != cudaSuccess) {
        gb_set_error("gb_kv4_attention_decode: launch failed: %s", cudaGetErrorString(rc));
        return 2;
    }
    if (blocks > 1) gb_launch(GB_PDL_ATTENTION, kv4_even_merge_kernel<HD>, dim3(blocks, group < KV4M_HEADS ? group : KV4M_HEADS), dim3(KV4E_GROUPS * HD / 4), 0, stream, a);
    return gb_check_launch("gb_kv4_attention_decode");
}

// 1 if the head size is one these kernels are built for.
GB_EXPORT int gb_kv4_attention_decode_supported(int hd) { return hd == 32 || hd == 64 || hd == 96 || hd == 128 || hd == 256; }

#define KV4M_CASE(HD_, call) \
    if (hd == HD_) return call;
#define KV4M_CASES(name, ...) \
    KV4M_CASE(32, name<32>(__VA_ARGS__)) KV4M_CASE(64, name<64>(__VA_ARGS__)) KV4M_CASE(96, name<96>(__VA_ARGS__)) KV4M_CASE(128, name<128>(__VA_ARGS__)) KV4M_CASE(256, name<256>(__VA_ARGS__))

// Blocks that gb_kv4_attention_decode may be given for even shares (0: none, the sizes are not built, or too many rows).
GB_EXPORT int gb_kv4_attention_decode_blocks(int n, int nh, int nkv, int hd, long long reach) {
    if (n <= 0 || n > KV4E_ROWS || nkv <= 0 || nh <= 0 || nh % nkv || reach <= 0) return 0;
    KV4M_CASES(kv4_even_blocks, n, nh, nkv, reach)
    return 0;
}

// As gb_kv4_attention_rows, q and out bfloat16. blocks == 0: the keys of a row in `cluster` (1, 2, 4 or 8) shares that are added up in a cluster. Else: even
// shares of all rows' keys among that many blocks, and parts float32 [2 * blocks * 8 * (hd + 2) + 4 * blocks], 16-byte aligned.
GB_EXPORT int gb_kv4_attention_decode(const void* q, long long q_stride, void* out, long long out_stride, const void* kcache, const void* vcache,
                                      const int* block_tables, int max_pages, const int* row_seq, const int* positions, int n, int nh, int nkv,
                                      int hd, int page_size, long long num_pages, float scale, int window, int cluster, int blocks, float* parts,
                                      int* status, cudaStream_t stream) {
    KV4_REQUIRE_SIZES("gb_kv4_attention_decode")
    GB_REQUIRE(n >= 0 && nh > 0 && nh % nkv == 0 && max_pages > 0, "gb_kv4_attention_decode: bad sizes (rows %d, heads %d of %d, tables of %d pages)", n, nh, nkv, max_pages);
    GB_REQUIRE(scale > 0.f && scale < INFINITY, "gb_kv4_attention_decode: scores must be scaled by a positive number");
    GB_REQUIRE(cluster == 1 || cluster == 2 || cluster == 4 || cluster == 8, "gb_kv4_attention_decode: clusters of %d are not built", cluster);
    GB_REQUIRE(blocks == 0 || (blocks > 0 && n <= KV4E_ROWS && parts != nullptr && (uintptr_t)parts % 16 == 0),
               "gb_kv4_attention_decode: even shares among %d blocks take up to %d rows and aligned scratch", blocks, KV4E_ROWS);
    GB_REQUIRE((long long)max_pages * page_size < (1ll << 31) - 64, "gb_kv4_attention_decode: block tables of %d pages reach too far", max_pages);
    GB_REQUIRE(n <= 65535 && nh <= 65535, "gb_kv4_attention_decode: %d rows of %d heads are too many for one launch", n, nh);
    GB_REQUIRE(((uintptr_t)kcache | (uintptr_t)vcache) % 16 == 0, "gb_kv4_attention_decode: the cache must be 16-byte aligned");
    GB_REQUIRE(num_pages * page_size / KV4_TILE * nkv < (1ll << 31), "gb_kv4_attention_decode: the pool has too many tiles");
    if (n == 0) return 0;
    Kv4AttnArgs a = {};
    a.q = q; a.q_stride = q_stride; a.out = out; a.out_stride = out_stride; a.kcache = (const unsigned char*)kcache;
    a.vcache = (const unsigned char*)vcache; a.block_tables = block_tables; a.max_pages = max_pages; a.row_seq = row_seq; a.positions = positions;
    a.n = n; a.nh = nh; a.nkv = nkv; a.hd = hd; a.page_size = page_size; a.num_pages = num_pages; a.scale = scale * KV4_LOG2E;
    a.window = window > 0 ? window : 0; a.parts = parts; a.status = status;
    KV4M_CASES(kv4_decode_launch, a, cluster, blocks, stream)
    GB_REQUIRE(false, "gb_kv4_attention_decode: head size %d is not built (32, 64, 96, 128, 256)", hd);
}
