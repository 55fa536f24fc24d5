// Attention of trees of drafted tokens over the paged cache on the 5th-generation tensor cores (sm_100a), bfloat16 at head sizes 64 and 128, without a window.
//
// A block has two units of 128 query rows (rows of the tree x query heads that share a key/value head; TMEM lanes). Where a request has at most 128 of them
// (SAME) both units have the same ones and take the tiles of 128 keys in turn, else they are 256 rows that take every tile. Either way two chains of
// scores -> softmax -> product keep tensor cores and exponentials busy in turn. Tiles of all items (request, key/value head, 256 or 128 rows) are cut evenly among
// one block a multiprocessor; a block goes through its pieces of items without draining its pipelines. An item that one block has whole is written out, the others'
// pieces go to the scratch, 32 rows side by side, and tree_tc_pieces_kernel adds up.
//   warp 0, 10  producers of keys and of values: a page is HD / 64 boxes of 64 channels, rings of stages in 128-byte-swizzled rows.
//   warp 1      issues S_g = Q_g K^T (M 128, N 128, K HD) and O_g += P_g V (M 128, N HD, K 128); the next scores of a unit right behind the product that reads P,
//               which lies over the first half of the scores' columns.
//   warps 2-9   softmax, four a unit, a row a thread; they lay the unit's queries out in shared memory, and write what comes out.
// Masks are looked at only in the tiles that reach into the tree (bits, 32 keys at a time). There values that are not finite numbers are taken out of shared
// memory, so that no weight of zero meets them; rows that see such a key get its part one key at a time.
// What bounds it: memory where rows are few (1 tree of 26 rows, 32/8 heads of 128, behind 131,071 tokens, 537 MB: 115 us, 4.7 TB/s; a longer context costs 6.6 TB/s
// of its keys, the rest is the first tiles, a piece's end and the launch that adds up), else a unit's chain (4 trees of 64 rows behind 8,000 to 16,001 tokens, 41 GFLOP:
// 78 us, 520 TFLOP/s). Every wait is bounded: a wait that runs out sets GB_STATUS_WAIT_TIMEOUT and the block winds down.
#include "tcgen05.cuh"
#include "tree_attention.cuh"

constexpr int TC5_M = 128, TC5_KEYS = 128, TC5_WARPS = 11, TC5_SEGS = 32;
constexpr int TC5_BLOCK = 128 * 128;      // bytes of 128 rows of 64 channels
constexpr float TC5_NEG_BIG = -1.0e30f;

template <int HD, bool SAME>
struct Tc5Shape {
    static constexpr int COLS = HD / 64, TILE = COLS * TC5_BLOCK;
    static constexpr int STAGES_K = HD == 128 ? 3 : SAME ? 6 : 5, STAGES_V = HD == 128 ? (SAME ? 3 : 2) : SAME ? 6 : 5;
    static constexpr int K_OFF = (SAME ? 1 : 2) * TILE, V_OFF = K_OFF + STAGES_K * TILE, SH_OFF = V_OFF + STAGES_V * TILE;
    static constexpr int O_COL = 2 * TC5_KEYS;
};

struct __align__(16) Tc5Shared {
    int4 seg[TC5_SEGS];                   // request, item of the request, first tile, tiles
    int piece[TC5_SEGS];
    float2 stat[2][TC5_M];                // (SAME) of a unit's row: maximum, sum
    uint64_t q_full;                      // softmax -> MMA: the queries of a piece lie in shared memory (and O of the one before has been read)
    uint64_t k_full[6], v_full[6], k_free[6], v_free[6];
    uint64_t s_full[2], p_most[2], p_ready[2], pv_done[2];
    long long at;                         // the tile of all items behind those of the list
    uint32_t tmem_base;
    int odd;                              // a value of the piece's tiles that reach into the tree is not a finite number
    int abort_flag, segs;                 // (segs: negative where the share ends with them)
    int issued[2], consumed[2];
};
static_assert(sizeof(Tc5Shared) <= 3 * 1024, "shared memory layout");

__device__ __forceinline__ uint64_t tc5_desc_mn(uint32_t smem_addr) {      // MN-major B operand: column blocks of 64 channels TC5_BLOCK bytes apart
    uint64_t d = 0;
    d |= (uint64_t)((smem_addr & 0x3FFFF) >> 4);
    d |= (uint64_t)((TC5_BLOCK >> 4) & 0x3FFF) << 16;
    d |= (uint64_t)(1024 >> 4) << 32;
    d |= (uint64_t)1 << 46;
    d |= (uint64_t)2 << 61;
    return d;
}
__device__ __forceinline__ float tc5_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float tc5_max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ void tc5_store16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr), "r"(r[0]), "r"(r[1]),
                 "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]),
                 "r"(r[14]), "r"(r[15])
                 : "memory");
}

// 16 channels of a row's O get the part of the keys from `k0` to `k1` whose values are not all finite, one at a time (they were taken out of the products).
template <int HD>
__device__ __forceinline__ void tree_odd_keys(const TreeArgs& a, const TreeSeq& s, int row, int m, int kvh, int G, int k0, int k1, float top, int c, uint32_t (&o)[16]) {
    const __nv_bfloat16* q = (const __nv_bfloat16*)a.q + (size_t)row * a.q_stride + (size_t)(kvh * G + m % G) * HD;
    const int pos = a.positions[row];
#pragma unroll 1
    for (int key = k0; key < k1; ++key) {
        const int page = s.page(a, key / a.page_size);
        if (page < 0 || !s.sees(a, row, pos, key)) continue;
        const size_t at = (((size_t)page * a.nkv + kvh) * a.page_size + key % a.page_size) * HD;
        const __nv_bfloat16* k = (const __nv_bfloat16*)a.kcache + at;
        const __nv_bfloat16* v = (const __nv_bfloat16*)a.vcache + at;
        float dot = 0.f;
        bool odd = false;
#pragma unroll 1
        for (int i = 0; i < HD; ++i) {
            dot = fmaf(__bfloat162float(q[i]), __bfloat162float(k[i]), dot);
            odd = odd || !isfinite(__bfloat162float(v[i]));
        }
        if (!odd) continue;
        const float p = tc5_exp2(dot * a.scale * 1.4426950408889634f - top);
#pragma unroll
        for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(fmaf(p, __bfloat162float(v[c + i]), __uint_as_float(o[i])));
    }
}

template <int HD, bool SAME>
__global__ void __launch_bounds__(TC5_WARPS * 32) tree_attention_tc_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                                                                           const TreeArgs a, int num_seqs, int page_shift) {
    using Sh = Tc5Shape<HD, SAME>;
    constexpr int SK = Sh::STAGES_K, SV = Sh::STAGES_V, COLS = Sh::COLS, ROWS = SAME ? TC5_M : 2 * TC5_M, P = HD + 2;
    extern __shared__ __align__(1024) unsigned char tc5_mem[];
    unsigned char* Qs = tc5_mem;
    unsigned char* Ks = tc5_mem + Sh::K_OFF;
    unsigned char* Vs = tc5_mem + Sh::V_OFF;
    Tc5Shared& sh = *reinterpret_cast<Tc5Shared*>(tc5_mem + Sh::SH_OFF);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, G = a.nh / a.nkv;
    gb_pdl_wait();
    gb_pdl_launch_dependents();
    if (smem_u32(tc5_mem) & 1023u) {              // swizzled tiles want 1024-byte alignment: refuse rather than compute nonsense
        if (tid == 0) atomicOr(a.status, GB_STATUS_WAIT_TIMEOUT);
        return;
    }
    // The next pieces of the block's share, up to TC5_SEGS, from tile `at` on (all of warp 0); count 0: there are none.
    auto list = [&](bool begin) {
        TreeCut cut(a, num_seqs, ROWS, TC5_KEYS, gridDim.x, TREE_LEAST_SHARE);
        const long long end = min(cut.total, (blockIdx.x + 1) * cut.share);
        long long at = begin ? min(cut.total, blockIdx.x * cut.share) : sh.at;
        int count = 0;
        if (at < end) cut.seek(at);
        for (; at < end && count < TC5_SEGS; ++count) {
            const TreeSeq s(a, cut.seq);
            const int all = s.tiles(TC5_KEYS);
            const long long off = at - cut.tile0;
            const int item = (int)(off / all), tile0 = (int)(off - (long long)item * all), tiles = (int)min((long long)all - tile0, end - at);
            if (lane == 0) {
                sh.seg[count] = make_int4(cut.seq, item, tile0, tiles);
                sh.piece[count] = (int)(cut.item0 + item + blockIdx.x);
            }
            at += tiles;
            if (at < end) cut.reach(at);
        }
        __syncwarp();
        if (lane == 0) { sh.segs = at < end ? count : -count; sh.at = at; }
    };
    if (warp == 0) {
        list(true);
    } else if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&sh.tmem_base)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    } else if (tid == 64) {
        mbar_init(&sh.q_full, 8);
        for (int b = 0; b < SK; ++b) { mbar_init(&sh.k_full[b], 1); mbar_init(&sh.k_free[b], 1); }
        for (int b = 0; b < SV; ++b) { mbar_init(&sh.v_full[b], 1); mbar_init(&sh.v_free[b], 1); }
        for (int g = 0; g < 2; ++g) {
            mbar_init(&sh.s_full[g], 1);
            mbar_init(&sh.pv_done[g], 1);
            mbar_init(&sh.p_most[g], 4);
            mbar_init(&sh.p_ready[g], 4);
        }
        sh.abort_flag = 0;
        sh.issued[0] = sh.issued[1] = sh.consumed[0] = sh.consumed[1] = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sh.tmem_base;
    volatile int* abort_flag = &sh.abort_flag;

    // what each role counts over all pieces
    int tiles_done = 0;                           // tiles of keys and values
    int pieces_done = 0, steps = 0, steps1 = 0;   // the issuer and the softmax: pieces, and their unit's tiles (the issuer: unit 0's and unit 1's)
    bool ok = true;
    while (true) {
        const bool more = sh.segs > 0;
        const int segs = abs(sh.segs);

        if (warp == 0 || warp == TC5_WARPS - 1) {
            // --------------------------------------------------------------------- producers
            const int what = warp == 0 ? 0 : 1, ppt = TC5_KEYS >> page_shift;      // pages per tile (1 .. 16), COLS boxes each
            uint64_t* full = what == 0 ? sh.k_full : sh.v_full;
            uint64_t* freed = what == 0 ? sh.k_free : sh.v_free;
            unsigned char* ring = what == 0 ? Ks : Vs;
            const CUtensorMap* map = what == 0 ? &map_k : &map_v;
            const int stages = what == 0 ? SK : SV, nowhere = (int)(a.num_pages * a.nkv * a.page_size);
            bool bad = false;
            for (int i = 0; i < segs && ok; ++i) {
                const int4 seg = sh.seg[i];
                const TreeSeq s(a, seg.x);
                const int kvh = seg.y / ((s.rows * G + ROWS - 1) / ROWS);
                // the first row of this lane's page of a tile (lanes COLS i .. have page i); one that is missing lies behind all pages, where a copy reads zeros
                auto row_of = [&](int tile) -> int {
                    const int index = ((tile * TC5_KEYS) >> page_shift) + lane / COLS;
                    if (lane >= COLS * ppt || (index << page_shift) >= s.length) return nowhere;
                    const long long page = s.page(a, index);
                    if (page >= 0) return (int)((page * a.nkv + kvh) * a.page_size);
                    bad = true;
                    return nowhere;
                };
                int row = row_of(seg.z);
                for (int j = 0; j < seg.w; ++j, ++tiles_done) {
                    const int st = tiles_done % stages, next_row = j + 1 < seg.w ? row_of(seg.z + j + 1) : nowhere;      // in flight during the wait
                    if (lane == 0 && tiles_done >= stages) ok = mbar_wait(&freed[st], (tiles_done / stages - 1) & 1, abort_flag, a.status);
                    ok = __shfl_sync(0xffffffffu, ok ? 1 : 0, 0) != 0;
                    if (!ok) break;
                    if (lane == 0) mbar_expect_tx(&full[st], Sh::TILE);
                    __syncwarp();
                    if (lane < COLS * ppt)
                        tma_load_2d(ring + st * Sh::TILE + lane % COLS * TC5_BLOCK + lane / COLS * a.page_size * 128, map, &full[st], lane % COLS * 64, row);
                    __syncwarp();
                    if (lane == 0) sh.issued[what] = tiles_done + 1;
                    row = next_row;
                }
            }
            if (bad && what == 0) atomicOr(a.status, GB_STATUS_BAD_SLOT);
        } else if (warp == 1) {
            // --------------------------------------------------------------------- MMA issuer
            const uint32_t idesc_qk = umma_idesc(TC5_M, TC5_KEYS), idesc_pv = umma_idesc(TC5_M, HD) | (1u << 16);   // (B of the second is MN-major)
            const uint64_t q_desc = umma_desc(smem_u32(Qs)), k_desc = umma_desc(smem_u32(Ks)), v_desc = tc5_desc_mn(smem_u32(Vs));
            for (int i = 0; i < segs && ok; ++i) {
                const int4 seg = sh.seg[i];
                int units = 2;
                if constexpr (!SAME) {
                    const TreeSeq s(a, seg.x);
                    const int pairs = (s.rows * G + ROWS - 1) / ROWS;
                    units = s.rows * G - seg.y % pairs * ROWS > TC5_M ? 2 : 1;
                }
                // steps: (tile, unit) in the order in which they are taken; in turn over the tiles, or both units of each
                const int n = SAME ? seg.w : seg.w * units, ahead = SAME ? 2 : units;
                if (elect_one()) {
                    auto tile_of = [&](int x) { return tiles_done + (SAME ? x : x / units); };
                    auto unit_of = [&](int x) { return SAME ? x & 1 : x % units; };
                    auto last_of = [&](int x) { return SAME || unit_of(x) == units - 1; };      // the last step that reads its tile
                    auto scores = [&](int x) {
                        const int tile = tile_of(x), g = unit_of(x), st = tile % SK;
                        if (SAME || unit_of(x) == 0) {
                            if (!mbar_wait(&sh.k_full[st], (tile / SK) & 1, abort_flag, a.status)) return false;
                            sh.consumed[0] = tile + 1;
                            tc_fence_after();
                        }
                        const uint64_t qd = q_desc + (uint64_t)((SAME ? 0 : g * Sh::TILE) >> 4), kd = k_desc + (uint64_t)((st * Sh::TILE) >> 4);
#pragma unroll
                        for (int k = 0; k < HD / 16; ++k) {
                            const uint64_t o = (uint64_t)((k / 4) * (TC5_BLOCK >> 4) + (k % 4) * 2);
                            umma_bf16(tmem + (uint32_t)(g * TC5_KEYS), qd + o, kd + o, idesc_qk, k ? 1u : 0u);
                        }
                        umma_commit(&sh.s_full[g]);
                        if (last_of(x)) umma_commit(&sh.k_free[st]);
                        return true;
                    };
                    ok = mbar_wait(&sh.q_full, pieces_done & 1, abort_flag, a.status);
                    if (ok) {
                        tc_fence_after();
                        for (int x = 0; x < ahead && x < n && ok; ++x) ok = scores(x);
                    }
                    for (int x = 0; x < n && ok; ++x) {
                        const int tile = tile_of(x), g = unit_of(x), st = tile % SV;
                        if (SAME || g == 0) {
                            ok = mbar_wait(&sh.v_full[st], (tile / SV) & 1, abort_flag, a.status);
                            if (!ok) break;
                            sh.consumed[1] = tile + 1;
                        }
                        const uint64_t vd = v_desc + (uint64_t)((st * Sh::TILE) >> 4);
                        const uint32_t pt = tmem + (uint32_t)(g * TC5_KEYS), ot = tmem + (uint32_t)(Sh::O_COL + g * HD);
                        const bool first = SAME ? x < 2 : x < units;      // the unit's first of the piece: O begins anew
                        const int step = g ? steps1 : steps;
                        ok = mbar_wait(&sh.p_most[g], step & 1, abort_flag, a.status);
                        if (!ok) break;
                        tc_fence_after();
#pragma unroll
                        for (int kk = 0; kk < 6; ++kk)      // 16 keys per instruction: 8 columns of P
                            umma_bf16_ts(ot, pt + (uint32_t)(kk * 8), vd + (uint64_t)(kk * 16 * 128 >> 4), idesc_pv, (first && kk == 0) ? 0u : 1u);
                        ok = mbar_wait(&sh.p_ready[g], step & 1, abort_flag, a.status);
                        if (!ok) break;
                        tc_fence_after();
#pragma unroll
                        for (int kk = 6; kk < 8; ++kk) umma_bf16_ts(ot, pt + (uint32_t)(kk * 8), vd + (uint64_t)(kk * 16 * 128 >> 4), idesc_pv, 1u);
                        umma_commit(&sh.pv_done[g]);
                        if (last_of(x)) umma_commit(&sh.v_free[st]);
                        if (g) ++steps1; else ++steps;
                        if (x + ahead < n) ok = scores(x + ahead);      // (over the unit's P, which the product just issued reads before)
                    }
                }
                ok = __all_sync(0xffffffffu, ok);
                steps = __reduce_max_sync(0xffffffffu, steps);      // (one lane has counted them)
                steps1 = __reduce_max_sync(0xffffffffu, steps1);
                tiles_done += seg.w;
                ++pieces_done;
            }
        } else {
            // --------------------------------------------------------------------- softmax
            const int q = warp & 3;                       // the quarter of TMEM lanes this warp may read
            const int g = (warp - 2) >> 2;                // the unit
            const int r = q * 32 + lane;                  // this thread's row of the unit
            const float sl2 = a.scale * 1.4426950408889634f;
            const uint32_t lane_base = tmem + ((uint32_t)(q * 32) << 16), s_col = (uint32_t)(g * TC5_KEYS), o_col = (uint32_t)(Sh::O_COL + g * HD);
            auto gave_up = [&]() {
                if (!__any_sync(0xffffffffu, *abort_flag)) return false;
                ok = false;
                return true;
            };
            for (int i = 0; i < segs; tiles_done += sh.seg[i].w, ++i) {
                int mine, units = 2;                      // tiles of this unit
                int before;                               // its tiles that all lie before the tree
                // both units are done with the piece before (every warp comes here for every piece, also one that has given up)
                asm volatile("barrier.cta.sync 1, 256;" ::: "memory");
                if (!ok) {
                    if constexpr (SAME) asm volatile("barrier.cta.sync 2, 256;" ::: "memory");
                    continue;
                }
                {
                    const int4 seg = sh.seg[i];
                    const TreeSeq s(a, seg.x);
                    const int M = s.rows * G, pairs = (M + ROWS - 1) / ROWS, m = seg.y % pairs * ROWS + (SAME ? 0 : g * TC5_M) + r;
                    if constexpr (!SAME) units = M - seg.y % pairs * ROWS > TC5_M ? 2 : 1;
                    mine = SAME ? (seg.w + 1 - g) / 2 : g < units ? seg.w : 0;
                    // the unit's queries into swizzled rows (zeros behind the last)
                    if (tid == 64) sh.odd = 0;
                    before = s.start / TC5_KEYS - seg.z;
                    before = SAME ? (before + 1 - g) / 2 : before;      // (negative where the piece begins behind: all are masked)
                    if (!SAME || g == 0) {
                        const uint4* from = reinterpret_cast<const uint4*>((const __nv_bfloat16*)a.q + (size_t)(s.row0 + m / G) * a.q_stride + (size_t)(seg.y / pairs * G + m % G) * HD);
                        unsigned char* to = Qs + (SAME ? 0 : g * Sh::TILE) + r * 128;
#pragma unroll
                        for (int c = 0; c < HD / 8; ++c)
                            *reinterpret_cast<uint4*>(to + c / 8 * TC5_BLOCK + ((c % 8) ^ (r & 7)) * 16) = m < M ? from[c] : make_uint4(0, 0, 0, 0);
                    }
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    tc_fence_before();                    // (O of the piece before has been read)
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&sh.q_full);
                }
                float m_run = TC5_NEG_BIG, l_run = 0.f;
                for (int j = 0; j < mine; ++j) {
                    if (!mbar_wait_warp(&sh.s_full[g], steps & 1, abort_flag, a.status)) { ok = false; break; }
                    tc_fence_after();
                    if (j >= before) {
                        const int4 seg = sh.seg[i];
                        const TreeSeq s(a, seg.x);
                        const int M = s.rows * G, m = seg.y % ((M + ROWS - 1) / ROWS) * ROWS + (SAME ? 0 : g * TC5_M) + r, row = m < M ? s.row0 + m / G : -1;
                        const int tile = seg.z + (SAME ? 2 * j + g : j), first_key = tile * TC5_KEYS;
                        // scores of keys that the row does not see become minus infinity where they lie
                        for (int w = 0; w < 4; ++w) {
                            const unsigned see = tree_bits(a, s.rows, row, first_key + 32 * w - s.start);
                            uint32_t part[32];
                            tmem_load32(lane_base + s_col + (uint32_t)(32 * w), part);
#pragma unroll
                            for (int k = 0; k < 32; ++k)
                                if (!(see >> k & 1u)) part[k] = 0xff800000u;
                            tmem_store32(lane_base + s_col + (uint32_t)(32 * w), part);
                        }
                        if (SAME || g == 0) {
                            // a key's values a thread; the product waits for this unit's weights, which come behind
                            const int ring = (tiles_done + tile - seg.z) % SV, use = (tiles_done + tile - seg.z) / SV;
                            if (!mbar_wait_warp(&sh.v_full[ring], use & 1, abort_flag, a.status)) { ok = false; break; }
                            unsigned char* v = Vs + ring * Sh::TILE + r * 128;
                            bool odd = false;
#pragma unroll
                            for (int c = 0; c < HD / 8; ++c) {
                                const uint4 x = *reinterpret_cast<const uint4*>(v + c / 8 * TC5_BLOCK + c % 8 * 16);      // (in whatever order)
                                const uint32_t w4[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                                for (int e = 0; e < 4; ++e) odd = odd || (w4[e] & 0x7f80u) == 0x7f80u || (w4[e] & 0x7f800000u) == 0x7f800000u;
                            }
                            if (odd) {
#pragma unroll
                                for (int c = 0; c < HD / 8; ++c) *reinterpret_cast<uint4*>(v + c / 8 * TC5_BLOCK + c % 8 * 16) = make_uint4(0, 0, 0, 0);
                                if (first_key + r < s.length) sh.odd = 1;
                            }
                            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                        }
                    }
                    // The scores of the last 64 keys stay in registers; the first 64 are read once more (all 128 beside the rest spill)
                    float mx4[4] = {TC5_NEG_BIG, TC5_NEG_BIG, TC5_NEG_BIG, TC5_NEG_BIG};
                    uint32_t sv[TC5_KEYS / 2];
#pragma unroll
                    for (int half = 0; half < TC5_KEYS; half += 64) {
                        tmem_load64(lane_base + s_col + (uint32_t)half, sv);
#pragma unroll
                        for (int k = 0; k < 64; k += 8)
#pragma unroll
                            for (int u = 0; u < 4; ++u) mx4[u] = tc5_max3(mx4[u], __uint_as_float(sv[k + 2 * u]), __uint_as_float(sv[k + 2 * u + 1]));
                    }
                    const float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3])) * sl2;
                    // the running maximum (in the exponent, base 2) rises, and O is rescaled, only when it is exceeded by more than 8
                    const bool raise = mx - m_run > 8.0f;
                    if (j == 0) {
                        if (raise) m_run = mx;
                    } else if (__any_sync(0xffffffffu, raise)) {
                        // the unit's product before is complete (these scores were issued behind it)
                        if (!mbar_wait_warp(&sh.pv_done[g], (steps - 1) & 1, abort_flag, a.status)) { ok = false; break; }
                        tc_fence_after();
                        const float corr = raise ? tc5_exp2(m_run - mx) : 1.0f;
                        if (raise) m_run = mx;
                        l_run *= corr;
#pragma unroll
                        for (int c = 0; c < HD; c += 16) {
                            uint32_t ov[16];
                            tmem_load16(lane_base + o_col + (uint32_t)c, ov);
#pragma unroll
                            for (int k = 0; k < 16; ++k) ov[k] = __float_as_uint(__uint_as_float(ov[k]) * corr);
                            tc5_store16(lane_base + o_col + (uint32_t)c, ov);
                        }
                    }
                    const float2 scale2 = make_float2(sl2, sl2), off2 = make_float2(-m_run, -m_run);
                    float2 l2[4] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f), make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
                    for (int part = 0; part < TC5_KEYS; part += 32) {
                        uint32_t pw[16], first[32];
                        if (part < 64) tmem_load32(lane_base + s_col + (uint32_t)part, first);      // (P lies over scores that have been read)
#pragma unroll
                        for (int c = 0; c < 32; c += 2) {
                            const uint32_t s0 = part < 64 ? first[c] : sv[(part + c) & 63], s1 = part < 64 ? first[c + 1] : sv[(part + c + 1) & 63];
                            const float2 y = __ffma2_rn(make_float2(__uint_as_float(s0), __uint_as_float(s1)), scale2, off2);
                            const float2 p = make_float2(tc5_exp2(y.x), tc5_exp2(y.y));
                            l2[(c >> 1) & 3] = __fadd2_rn(l2[(c >> 1) & 3], p);
                            pw[c >> 1] = pack2(__float_as_uint(p.x), __float_as_uint(p.y));
                        }
                        tc5_store16(lane_base + s_col + (uint32_t)(part / 2), pw);
                        if (part == 64 && gave_up()) break;
                        if (part >= 64) {      // three quarters, and the rest
                            asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                            tc_fence_before();
                            __syncwarp();
                            if (lane == 0) mbar_arrive(part == 64 ? &sh.p_most[g] : &sh.p_ready[g]);
                            if (part == 64 && gave_up()) break;
                        }
                    }
                    if (!ok) break;
                    const float2 lsum = __fadd2_rn(__fadd2_rn(l2[0], l2[1]), __fadd2_rn(l2[2], l2[3]));
                    l_run += lsum.x + lsum.y;
                    ++steps;
                }
                if (ok && mine > 0) ok = mbar_wait_warp(&sh.pv_done[g], (steps - 1) & 1, abort_flag, a.status);
                // A row's result: O, relative to its maximum `top` (base 2), and the sum of its weights. SAME: the two units' parts are added up, each thread has half
                // of the row's channels of both, whose columns all warps of the row's lanes can read. (Every warp meets that barrier for every piece.)
                float top = m_run, l = l_run, f0 = 1.0f, f1 = 0.f;
                int from_c = 0, to_c = HD;
                const bool both = SAME && sh.seg[i].w > 1;      // (unit 0 has a tile always)
                if constexpr (SAME) {
                    sh.stat[g][r] = mine > 0 ? make_float2(m_run, l_run) : make_float2(-INFINITY, 0.f);
                    tc_fence_before();
                    asm volatile("barrier.cta.sync 2, 256;" ::: "memory");
                    const float2 s0 = sh.stat[0][r], s1 = sh.stat[1][r];
                    top = fmaxf(s0.x, s1.x);
                    f0 = tc5_exp2(s0.x - top);
                    f1 = both ? tc5_exp2(s1.x - top) : 0.f;
                    l = fmaf(s1.y, f1, s0.y * f0);
                    from_c = g * (HD / 2);
                    to_c = from_c + HD / 2;
                    if (__any_sync(0xffffffffu, *abort_flag)) ok = false;
                }
                if (!ok) continue;
                tc_fence_after();
                const int4 seg = sh.seg[i];
                const TreeSeq s(a, seg.x);
                const int M = s.rows * G, pairs = (M + ROWS - 1) / ROWS, kvh = seg.y / pairs, m = seg.y % pairs * ROWS + (SAME ? 0 : g * TC5_M) + r, row = m < M ? s.row0 + m / G : -1;
                const bool whole = seg.z == 0 && seg.w == s.tiles(TC5_KEYS);
                const float inv = l != 0.f ? 1.0f / l : 0.f;
                float* part = a.parts + ((size_t)sh.piece[i] * (SAME ? 1 : 2) + (SAME ? 0 : g)) * (TC5_M * P) + (size_t)q * (32 * P) + lane;
                __nv_bfloat16* dst = (__nv_bfloat16*)a.out + (size_t)(row < 0 ? 0 : row) * a.out_stride + (size_t)(kvh * G + m % G) * HD;
                for (int c = from_c; c < to_c; c += 16) {
                    uint32_t o[16];
                    if (SAME || mine > 0) tmem_load16(lane_base + (uint32_t)(Sh::O_COL + (SAME ? 0 : g * HD) + c), o);
                    else
#pragma unroll
                        for (int k = 0; k < 16; ++k) o[k] = 0u;
                    if constexpr (SAME) {
                        if (both) {
                            uint32_t o1[16];
                            tmem_load16(lane_base + (uint32_t)(Sh::O_COL + HD + c), o1);
#pragma unroll
                            for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(fmaf(__uint_as_float(o1[k]), f1, __uint_as_float(o[k]) * f0));
                        }
                    }
                    if (sh.odd && row >= 0) tree_odd_keys<HD>(a, s, row, m, kvh, G, max(seg.z, s.start / TC5_KEYS) * TC5_KEYS, min(s.length, (seg.z + seg.w) * TC5_KEYS), top, c, o);
                    if (whole) {
                        if (row >= 0) {
#pragma unroll
                            for (int k = 0; k < 16; k += 8) {
                                uint4 w;
                                w.x = pack2(__float_as_uint(__uint_as_float(o[k]) * inv), __float_as_uint(__uint_as_float(o[k + 1]) * inv));
                                w.y = pack2(__float_as_uint(__uint_as_float(o[k + 2]) * inv), __float_as_uint(__uint_as_float(o[k + 3]) * inv));
                                w.z = pack2(__float_as_uint(__uint_as_float(o[k + 4]) * inv), __float_as_uint(__uint_as_float(o[k + 5]) * inv));
                                w.w = pack2(__float_as_uint(__uint_as_float(o[k + 6]) * inv), __float_as_uint(__uint_as_float(o[k + 7]) * inv));
                                *reinterpret_cast<uint4*>(dst + c + k) = w;
                            }
                        }
                    } else {
#pragma unroll
                        for (int k = 0; k < 16; ++k) part[(c + k) * 32] = __uint_as_float(o[k]);
                    }
                }
                if (!whole && from_c == 0) {
                    part[HD * 32] = SAME || mine > 0 ? top : -INFINITY;
                    part[HD * 32 + 32] = l;
                }
            }
        }
        if (!more) break;
        __syncthreads();                          // (the list has been read)
        if (*abort_flag) break;
        if (warp == 0) list(false);
        __syncthreads();
    }

    // padding requests' rows are zeros
    for (int seq = blockIdx.x; seq < num_seqs; seq += gridDim.x) {
        if (a.start_pos[seq] >= 0) continue;
        const TreeSeq s(a, seq);
        for (int i = tid; i < s.rows * a.nh * (HD / 2); i += TC5_WARPS * 32)
            *reinterpret_cast<uint32_t*>((__nv_bfloat16*)a.out + (size_t)(s.row0 + i / (a.nh * (HD / 2))) * a.out_stride + i % (a.nh * (HD / 2)) * 2) = 0u;
    }
    // ------------------------------------------------------------------------------- wind down
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        if (lane == 0 && sh.abort_flag) {
            // copies that were issued but never consumed may still be in flight: wait for them (bounded)
            for (int what = 0; what < 2; ++what)
                for (int it = sh.consumed[what]; it < sh.issued[what]; ++it) {
                    const int stages = what == 0 ? SK : SV;
                    uint64_t* bar = what == 0 ? &sh.k_full[it % stages] : &sh.v_full[it % stages];
                    const long long t1 = clock64();
                    while (!mbar_try_wait(bar, (it / stages) & 1) && clock64() - t1 < TC_WAIT_CYCLES) {}
                }
        }
        __syncwarp();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
    }
}

// Adds up the pieces of items that several blocks share: EACH rows of a unit a block (x: rows and item, y: request). A thread has four rows of a channel.
template <int HD, bool SAME, int EACH>
__global__ void __launch_bounds__(256) tree_tc_pieces_kernel(const TreeArgs a, int num_seqs, int pairs_most, int blocks) {
    constexpr int P = HD + 2, ROWS = SAME ? TC5_M : 2 * TC5_M, BATCH = 8, GROUPS = ROWS / EACH, QUADS = EACH / 4, LANES = 256 / EACH;
    __shared__ float2 stats[EACH];                // of a row: maximum, 1 / sum
    __shared__ float sums[EACH][HD + 1];
    gb_pdl_launch_dependents();
    gb_pdl_wait();
    const int seq = blockIdx.y, G = a.nh / a.nkv, group = blockIdx.x % GROUPS, pair = blockIdx.x / GROUPS % pairs_most, kvh = blockIdx.x / GROUPS / pairs_most, tid = threadIdx.x;
    const TreeSeq s(a, seq);
    const int M = s.rows * G, m0 = pair * ROWS + group * EACH;
    if (s.start < 0 || m0 >= M) return;
    TreeCut cut(a, num_seqs, ROWS, TC5_KEYS, blocks, TREE_LEAST_SHARE);
    cut.seek_seq(seq);
    const int all = s.tiles(TC5_KEYS), item = kvh * ((M + ROWS - 1) / ROWS) + pair;
    const long long t0 = cut.tile0 + (long long)item * all, b0 = t0 / cut.share;
    const int count = (int)((t0 + all - 1) / cut.share - b0) + 1;
    if (count == 1) return;
    constexpr int STEP = ROWS * P;
    const int u0 = group * EACH;                  // of the first row in the item
    const float* first = a.parts + (size_t)(cut.item0 + item + b0) * STEP + u0 / 32 * (32 * P) + u0 % 32;
    {
        const int r = tid / LANES;
        const float* from = first + HD * 32 + r;
        float top = -INFINITY, l = 0.f;
        for (int b = tid % LANES; b < count; b += LANES) {
            const float m = from[(size_t)b * STEP], up = fmaxf(top, m), o = up == -INFINITY ? 0.f : up;
            l = l * tc5_exp2(top - o) + from[(size_t)b * STEP + 32] * tc5_exp2(m - o);
            top = up;
        }
        float most = top;
#pragma unroll
        for (int o = 1; o < LANES; o <<= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
        const float o = most == -INFINITY ? 0.f : most;
        l *= tc5_exp2(top - o);
#pragma unroll
        for (int k = 1; k < LANES; k <<= 1) l += __shfl_xor_sync(0xffffffffu, l, k);
        if (tid % LANES == 0) stats[r] = make_float2(o, l != 0.f ? 1.0f / l : 0.f);
    }
    __syncthreads();
    for (int i = tid; i < QUADS * HD; i += 256) {
        const int r = i % QUADS * 4, c = i / QUADS;
        float top[4], sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < 4; ++k) top[k] = stats[r + k].x;
        const float* from = first + r;
        for (int b = 0; b < count; b += BATCH) {
            float4 v[BATCH], m[BATCH];
#pragma unroll
            for (int u = 0; u < BATCH; ++u) {
                const float* at = from + (size_t)min(b + u, count - 1) * STEP;
                v[u] = *reinterpret_cast<const float4*>(at + c * 32);
                m[u] = *reinterpret_cast<const float4*>(at + HD * 32);
            }
#pragma unroll
            for (int u = 0; u < BATCH; ++u)
                if (b + u < count) {
                    sum[0] = fmaf(v[u].x, tc5_exp2(m[u].x - top[0]), sum[0]);
                    sum[1] = fmaf(v[u].y, tc5_exp2(m[u].y - top[1]), sum[1]);
                    sum[2] = fmaf(v[u].z, tc5_exp2(m[u].z - top[2]), sum[2]);
                    sum[3] = fmaf(v[u].w, tc5_exp2(m[u].w - top[3]), sum[3]);
                }
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) sums[r + k][c] = sum[k] * stats[r + k].y;
    }
    __syncthreads();
    for (int i = tid; i < EACH * (HD / 2); i += 256) {
        const int r = i / (HD / 2), c = i % (HD / 2) * 2, m = m0 + r;
        if (m >= M) break;
        *reinterpret_cast<uint32_t*>((__nv_bfloat16*)a.out + (size_t)(s.row0 + m / G) * a.out_stride + (kvh * G + m % G) * HD + c) =
            pack2(__float_as_uint(sums[r][c]), __float_as_uint(sums[r][c + 1]));
    }
}

template <int HD, bool SAME>
static int tc5_launch(const TreeArgs& a, int blocks, int num_seqs, int max_rows, cudaStream_t stream) {
    using Sh = Tc5Shape<HD, SAME>;
    constexpr int SMEM = Sh::SH_OFF + (int)sizeof(Tc5Shared);
    static_assert(SMEM <= 227 * 1024, "the block does not fit");
    CUtensorMap mk, mv;
    if (tc_make_map_2d(&mk, a.kcache, a.num_pages * a.nkv * a.page_size, HD, HD, a.page_size, 64, "gb_tree_attention")) return 1;
    if (tc_make_map_2d(&mv, a.vcache, a.num_pages * a.nkv * a.page_size, HD, HD, a.page_size, 64, "gb_tree_attention")) return 1;
    cudaError_t e = cudaFuncSetAttribute(tree_attention_tc_kernel<HD, SAME>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM);
    GB_REQUIRE(e == cudaSuccess, "gb_tree_attention: %d bytes of shared memory refused: %s", SMEM, cudaGetErrorString(e));
    int page_shift = 0;
    while ((1 << page_shift) < a.page_size) ++page_shift;
    e = gb_launch(GB_PDL_ATTENTION, tree_attention_tc_kernel<HD, SAME>, dim3(blocks), dim3(TC5_WARPS * 32), SMEM, stream, mk, mv, a, num_seqs, page_shift);
    GB_REQUIRE(e == cudaSuccess, "gb_tree_attention: launch failed: %s", cudaGetErrorString(e));
    const int rows = SAME ? TC5_M : 2 * TC5_M, pairs = gb_ceil_div((long long)max_rows * (a.nh / a.nkv), rows);
    // 8 rows a block, else 32, where that leaves few of them: 1 tree of 64 rows, 32/8 heads of 128, behind 5,800 tokens 43 and 45 us, 4 behind 12,000 89 and 80
    const bool fine = (long long)pairs * a.nkv * num_seqs * (rows / 8) <= 4 * 148;
    const dim3 grid(pairs * a.nkv * (rows / (fine ? 8 : 32)), num_seqs);
    e = gb_launch(GB_PDL_ATTENTION, fine ? tree_tc_pieces_kernel<HD, SAME, 8> : tree_tc_pieces_kernel<HD, SAME, 32>, grid, dim3(256), 0, stream, a, num_seqs, pairs, blocks);
    GB_REQUIRE(e == cudaSuccess, "gb_tree_attention: launch failed: %s", cudaGetErrorString(e));
    return gb_check_launch("gb_tree_attention");
}

int gb_tree_attention_tc(const TreeArgs& a, const TreePlan& plan, int num_seqs, int max_rows, cudaStream_t stream) {
    GB_REQUIRE(a.num_pages * a.nkv * a.page_size < (1ll << 31), "gb_tree_attention: the pages hold too many rows");
    if (a.hd == 64) return plan.same ? tc5_launch<64, true>(a, plan.blocks, num_seqs, max_rows, stream) : tc5_launch<64, false>(a, plan.blocks, num_seqs, max_rows, stream);
    return plan.same ? tc5_launch<128, true>(a, plan.blocks, num_seqs, max_rows, stream) : tc5_launch<128, false>(a, plan.blocks, num_seqs, max_rows, stream);
}
