// Causal grouped-query flash attention for prompt portions at head size 128 on the 5th-generation tensor cores (sm_100a), over pages of
// bfloat16. The scheme is attention_prefill_tc.cu's (head size 64), laid out for twice the channels:
//
// One block = two units that share a head of keys and values, over tiles of 128 keys; a unit is 128 consecutive query rows of one request for one
// query head. (Units of a key/value head are counted over its query heads first, then over the rows, so that a pair covers nearly the same keys: at an
// odd number of query heads a key/value head some pairs straddle two row tiles, and run over the union of what the two need.)
//   warp 0, 10  producers of keys (and the query tiles, once) and of values: a page is two boxes of 64 channels, each issued by a lane of its own,
//               into rings of three and two stages (two 128-byte-swizzled column blocks a tile, 32 KB).
//   warp 1      issues S_gj = Q_g K_j^T (M 128, N 128, K 128) into TMEM columns 128 g and O_g += P_gj V_j (M 128, N 128, K 128), unit g = 0, 1.
//   warps 2-9   softmax, four warps a unit. A thread owns a row (a TMEM lane). P, rounded to bfloat16, goes back over the first half of S's own
//               columns: two score buffers and two accumulators of 128 columns fill the 512 that there are, so there is no room for P beside
//               them. The tensor core works in the order of issue, so the unit's next scores are issued right behind the product that reads P;
//               that product starts on the first 96 keys' weights while the last 32 are formed.
// What bounds it: a unit's chain of scores, softmax and weighted sum, each of which waits for the one before. Per unit and tile the two products are
// 1,024 cycles of the tensor core and the 16,384 exponentials as many of the unit that forms them; the two units keep both busy in turn. One
// unit a block (its key tiles in two interleaved chains) took 137 us with the unpacking below where this took 113: a tile of keys and values is 64 KB,
// and 148 blocks at one in 1,024 cycles each want more than the L2 cache hands out.
// The mask is applied only in tiles that cross a boundary; key tiles that no row sees are skipped. Zeros stand in the place of pages that no row of the
// block sees (behind its last row, before its window) or that are missing, so that P = 0 meets numbers whatever lies in other pages.
// Where blocks are few, a cluster of two or four shares a pair's key tiles; each block leaves O, maxima and sums in its shared memory, over what it has
// read, and adds up and writes its part of the channels from all of theirs.
// Every wait is bounded: a wait that runs out sets GB_STATUS_WAIT_TIMEOUT and the block winds down (waits for its own copies, frees its TMEM,
// returns). TMA loads use no multicast.
// Measured (2,048 rows behind 2,048 tokens, 32/8 heads, with the unpacking of 7 us): mma.sync 751 us, this kernel 107.
#include "tcgen05.cuh"

constexpr int AL_HD = 128, AL_BM = 128, AL_BN = 128, AL_KSTAGES = 3, AL_VSTAGES = 2, AL_WARPS = 11;
constexpr int AL_BLOCK = 128 * 128;                     // bytes of 128 rows of 64 channels
constexpr int AL_TILE = 2 * AL_BLOCK;
constexpr int AL_K_OFF = 2 * AL_TILE, AL_V_OFF = AL_K_OFF + AL_KSTAGES * AL_TILE, AL_SH_OFF = AL_V_OFF + AL_VSTAGES * AL_TILE;
constexpr int AL_SMEM = AL_SH_OFF + 512;
constexpr int AL_O_COL = 2 * AL_BN, AL_TMEM_COLS = 512;
constexpr float AL_NEG_BIG = -1.0e30f;
constexpr int AL_MAX_CLUSTER = 4;
constexpr int AL_STAT_OFF = 2 * AL_BM * AL_HD * 4;      // behind the two units' O as float32
static_assert(AL_STAT_OFF + 2 * 2 * AL_BM * 4 <= AL_SH_OFF, "a block's results lie over its queries and keys");
static_assert(AL_SMEM <= 227 * 1024 && AL_O_COL + 2 * AL_HD <= AL_TMEM_COLS, "the block does not fit");

struct __align__(8) AlShared {
    uint64_t q_full;
    uint64_t k_full[AL_KSTAGES], v_full[AL_VSTAGES];     // TMA -> MMA
    uint64_t s_full[2][AL_KSTAGES];  // MMA -> softmax and the keys' producer: the unit's scores of a tile are complete (by the keys' stage)
    uint64_t p_most[2], p_ready[2];  // softmax -> MMA: three quarters of the unit's P are in their place (and O is rescaled), all of it
    uint64_t pv_done[2][AL_VSTAGES]; // MMA -> softmax and the values' producer: O += P V is complete (by the values' stage)
    uint32_t tmem_base;
    int abort_flag;
    int issued[2], consumed[2], q_issued;
};
static_assert(sizeof(AlShared) <= 512, "shared memory layout");

// MN-major B operand (rows are keys, a head's channels contiguous) in 128-byte-swizzled rows: groups of eight keys 1024 bytes apart, column blocks
// of 64 channels lbo bytes apart.
__device__ __forceinline__ uint64_t al_desc_mn(uint32_t smem_addr, uint32_t lbo_bytes) {
    uint64_t d = 0;
    d |= (uint64_t)((smem_addr & 0x3FFFF) >> 4);
    d |= (uint64_t)((lbo_bytes >> 4) & 0x3FFF) << 16;
    d |= (uint64_t)(1024 >> 4) << 32;
    d |= (uint64_t)1 << 46;
    d |= (uint64_t)2 << 61;
    return d;
}
__device__ __forceinline__ float al_max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ float al_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// 16 of a thread's weights, rounded to bfloat16, to eight columns of its TMEM lane; the caller waits for the stores.
__device__ __forceinline__ void al_store16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr), "r"(r[0]), "r"(r[1]),
                 "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]),
                 "r"(r[14]), "r"(r[15])
                 : "memory");
}

// Four channels of a unit's row of O, in an order that keeps the rows of a warp in different banks.
__device__ __forceinline__ int al_piece(int g, int row, int four) { return ((g * AL_BM + row) * (AL_HD / 4) + (four ^ (row & 31))) * 16; }
__device__ __forceinline__ void al_cluster_sync() { asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ uint32_t al_peer_address(const void* own, int block) {      // where a block of the cluster has what lies here at `own`
    uint32_t p;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(p) : "r"(smem_u32(own)), "r"(block));
    return p;
}
__device__ __forceinline__ float al_peer(const void* own, int block) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(al_peer_address(own, block)) : "memory");
    return v;
}
__device__ __forceinline__ float4 al_peer4(const void* own, int block) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(al_peer_address(own, block)) : "memory");
    return v;
}

// CLUSTERS: the blocks of a cluster share a pair's keys. (One form for both costs the other registers: 108.5 us of 107.)
template <bool CLUSTERS>
__global__ void __launch_bounds__(AL_WARPS * 32) attention_prefill_128_kernel(
    const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
    __nv_bfloat16* __restrict__ out, long long out_stride, const int* __restrict__ block_tables, int max_pages, const int* __restrict__ seq_first_row,
    const int* __restrict__ seq_start_pos, int nh, int nkv, int page_size, int page_shift, long long num_pages, float scale, int window,
    int* __restrict__ status) {
    extern __shared__ __align__(1024) unsigned char al_smem[];
    unsigned char* Qs = al_smem;
    unsigned char* Ks = al_smem + AL_K_OFF;
    unsigned char* Vs = al_smem + AL_V_OFF;
    AlShared& sh = *reinterpret_cast<AlShared*>(al_smem + AL_SH_OFF);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    gb_pdl_wait();
    gb_pdl_launch_dependents();
    const int cluster = CLUSTERS ? gridDim.x / nkv : 1, kvh = blockIdx.x / cluster, rank = blockIdx.x % cluster;      // (all that returns early does so for a whole cluster)
    const int seq = blockIdx.y, group = nh / nkv, u0 = 2 * ((int)gridDim.z - 1 - (int)blockIdx.z);      // (the longest blocks start first)
    const int row0 = seq_first_row[seq], nrows = seq_first_row[seq + 1] - row0;
    const int q_lo0 = u0 / group * AL_BM, q_lo1 = (u0 + 1) / group * AL_BM;
    if (q_lo0 >= nrows) return;                   // uniform for the block, before anything is allocated
    const int units = q_lo1 < nrows ? 2 : 1;
    if (smem_u32(al_smem) & 1023u) {              // swizzled tiles want 1024-byte alignment: refuse rather than compute nonsense
        if (tid == 0) atomicOr(status, GB_STATUS_WAIT_TIMEOUT);
        return;
    }
    const int start_pos = seq_start_pos[seq];
    if (start_pos < 0) {                          // a padding request: its rows read as zeros downstream
        for (int g = 0; g < units && rank == 0; ++g) {
            const int lo = g ? q_lo1 : q_lo0, rows = min(AL_BM, nrows - lo), head = kvh * group + (u0 + g) % group;
            for (int i = tid; i < rows * (AL_HD / 8); i += blockDim.x)
                *reinterpret_cast<uint4*>(out + (size_t)(row0 + lo + i / (AL_HD / 8)) * out_stride + (size_t)head * AL_HD + i % (AL_HD / 8) * 8) = make_uint4(0, 0, 0, 0);
        }
        return;
    }
    const int* table = block_tables + (size_t)seq * max_pages;
    const int pos_hi = start_pos + min(nrows, (units == 2 ? q_lo1 : q_lo0) + AL_BM) - 1;
    const int key_lo = gb_first_key(start_pos + q_lo0, window), all_tiles = pos_hi / AL_BN - key_lo / AL_BN + 1;
    auto share = [&](int of) { return (int)((long long)all_tiles * of / cluster); };      // where the tiles of the cluster's block `of` begin
    const int kt_begin = key_lo / AL_BN + share(rank), total = share(rank + 1) - share(rank);

    if (tid == 0) {
        mbar_init(&sh.q_full, 1);
        for (int b = 0; b < AL_KSTAGES; ++b) mbar_init(&sh.k_full[b], 1);
        for (int b = 0; b < AL_VSTAGES; ++b) mbar_init(&sh.v_full[b], 1);
        for (int g = 0; g < 2; ++g) {
            for (int b = 0; b < AL_KSTAGES; ++b) mbar_init(&sh.s_full[g][b], 1);
            for (int b = 0; b < AL_VSTAGES; ++b) mbar_init(&sh.pv_done[g][b], 1);
            mbar_init(&sh.p_most[g], 4);
            mbar_init(&sh.p_ready[g], 4);
        }
        sh.abort_flag = 0;
        sh.issued[0] = sh.issued[1] = sh.consumed[0] = sh.consumed[1] = sh.q_issued = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh.tmem_base)), "r"(AL_TMEM_COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sh.tmem_base;
    volatile int* abort_flag = &sh.abort_flag;

    if (warp == 0 || warp == AL_WARPS - 1) {
        // ------------------------------------------------------------------------- producers
        const int what = warp == 0 ? 0 : 1;
        const int ppt = AL_BN >> page_shift;      // pages per key tile (1 .. 16), two boxes each
        uint64_t* full = what == 0 ? sh.k_full : sh.v_full;
        unsigned char* ring = what == 0 ? Ks : Vs;
        const CUtensorMap* map = what == 0 ? &map_k : &map_v;
        const int nowhere = (int)(num_pages * nkv * page_size);
        int bad = 0;
        if (what == 0 && lane == 0 && total > 0) {
            mbar_expect_tx(&sh.q_full, units * AL_TILE);
            for (int g = 0; g < units; ++g) {
                const int head = kvh * group + (u0 + g) % group, row = row0 + (g ? q_lo1 : q_lo0);
                tma_load_2d(Qs + g * AL_TILE, &map_q, &sh.q_full, head * AL_HD, row);
                tma_load_2d(Qs + g * AL_TILE + AL_BLOCK, &map_q, &sh.q_full, head * AL_HD + 64, row);
            }
            sh.q_issued = 1;
        }
        // The first row of this lane's page of key tile kt (lanes 2 i and 2 i + 1 have page i). A page that no row of the block sees, or that is missing,
        // lies behind all pages, where a copy reads zeros: what other requests, or earlier steps, left in a page must not meet a weight of zero.
        auto row_of = [&](int kt) -> int {
            const int pi = ((kt * AL_BN) >> page_shift) + (lane >> 1), first = pi << page_shift;
            if (lane >= 2 * ppt || first > pos_hi || first + page_size <= key_lo) return nowhere;
            const long long page = pi < max_pages ? table[pi] : -1;
            if (page >= 0 && page < num_pages) return (int)((page * nkv + kvh) * page_size);
            bad = 1;
            return nowhere;
        };
        int row = total > 0 ? row_of(kt_begin) : nowhere;
        for (int j = 0; j < total; ++j) {
            const int s = what == 0 ? j % AL_KSTAGES : j % AL_VSTAGES;
            const int next_row = j + 1 < total ? row_of(kt_begin + j + 1) : nowhere;      // in flight during the wait
            int ok = 1;
            if (lane == 0) {      // a stage is free when the last product of the tile that was in it is done
                if (what == 0 && j >= AL_KSTAGES) ok = mbar_wait(&sh.s_full[units - 1][s], (j / AL_KSTAGES - 1) & 1, abort_flag, status) ? 1 : 0;
                if (what == 1 && j >= AL_VSTAGES) ok = mbar_wait(&sh.pv_done[units - 1][s], (j / AL_VSTAGES - 1) & 1, abort_flag, status) ? 1 : 0;
            }
            ok = __shfl_sync(0xffffffffu, ok, 0);
            if (!ok) break;
            if (lane == 0) mbar_expect_tx(&full[s], AL_TILE);
            __syncwarp();
            if (lane < 2 * ppt)
                tma_load_2d(ring + s * AL_TILE + (lane & 1) * AL_BLOCK + (lane >> 1) * page_size * 128, map, &full[s], (lane & 1) * 64, row);
            __syncwarp();
            if (lane == 0) sh.issued[what] = j + 1;
            row = next_row;
        }
        if (bad && what == 0) atomicOr(status, GB_STATUS_BAD_SLOT);
    } else if (warp == 1) {
        // ------------------------------------------------------------------------- MMA issuer
        if (total > 0 && elect_one()) {
            const uint32_t idesc_qk = umma_idesc(AL_BM, AL_BN), idesc_pv = umma_idesc(AL_BM, AL_HD) | (1u << 16);   // (B of the second is MN-major)
            const uint64_t q_desc = umma_desc(smem_u32(Qs)), k_desc = umma_desc(smem_u32(Ks)), v_desc = al_desc_mn(smem_u32(Vs), AL_BLOCK);
            // What a step needs is waited for first; then the last of its weighted sum and the next scores are issued back to back.
            bool ok = mbar_wait(&sh.q_full, 0, abort_flag, status);
            int seen_k = 0, seen_v = 0;
            auto scores = [&](int g, int j) {
                const uint64_t qd = q_desc + (uint64_t)((g * AL_TILE) >> 4), kd = k_desc + (uint64_t)(((j % AL_KSTAGES) * AL_TILE) >> 4);
#pragma unroll
                for (int k = 0; k < AL_HD / 16; ++k) {
                    const uint64_t at = (uint64_t)((k / 4) * (AL_BLOCK >> 4) + (k % 4) * 2);
                    umma_bf16(tmem + (uint32_t)(g * AL_BN), qd + at, kd + at, idesc_qk, k ? 1u : 0u);
                }
                umma_commit(&sh.s_full[g][j % AL_KSTAGES]);
            };
            auto keys = [&](int j) {
                if (!mbar_wait(&sh.k_full[j % AL_KSTAGES], (j / AL_KSTAGES) & 1, abort_flag, status)) return false;
                seen_k = j + 1;
                return true;
            };
            if (ok) ok = keys(0);
            if (ok) {
                tc_fence_after();
                for (int g = 0; g < units; ++g) scores(g, 0);
            }
            for (int j = 0; ok && j < total; ++j) {
                if (j + 1 < total) ok = keys(j + 1);
                if (ok) ok = mbar_wait(&sh.v_full[j % AL_VSTAGES], (j / AL_VSTAGES) & 1, abort_flag, status);
                if (!ok) break;
                seen_v = j + 1;
                const uint64_t vd = v_desc + (uint64_t)(((j % AL_VSTAGES) * AL_TILE) >> 4);
                for (int g = 0; g < units; ++g) {
                    const uint32_t pt = tmem + (uint32_t)(g * AL_BN), ot = tmem + (uint32_t)(AL_O_COL + g * AL_HD);
                    ok = mbar_wait(&sh.p_most[g], j & 1, abort_flag, status);
                    if (!ok) break;
                    tc_fence_after();
#pragma unroll
                    for (int kk = 0; kk < 6; ++kk)      // 16 keys per instruction: 8 columns of P
                        umma_bf16_ts(ot, pt + (uint32_t)(kk * 8), vd + (uint64_t)(kk * 16 * 128 >> 4), idesc_pv, (j || kk) ? 1u : 0u);
                    ok = mbar_wait(&sh.p_ready[g], j & 1, abort_flag, status);
                    if (!ok) break;
                    tc_fence_after();
#pragma unroll
                    for (int kk = 6; kk < 8; ++kk) umma_bf16_ts(ot, pt + (uint32_t)(kk * 8), vd + (uint64_t)(kk * 16 * 128 >> 4), idesc_pv, 1u);
                    umma_commit(&sh.pv_done[g][j % AL_VSTAGES]);
                    if (j + 1 < total) scores(g, j + 1);      // (over the unit's P, which the product just issued reads before)
                }
            }
            sh.consumed[0] = seen_k;
            sh.consumed[1] = seen_v;
        }
    } else if ((warp - 2) >> 2 < units) {
        // ------------------------------------------------------------------------- softmax
        const int q = warp & 3;                        // the quarter of TMEM lanes this warp may read
        const int g = (warp - 2) >> 2;                 // the unit
        const int r = q * 32 + lane;                   // this thread's query row within the tile
        const float sl2 = scale * 1.4426950408889634f;
        const uint32_t lane_base = tmem + ((uint32_t)(q * 32) << 16), s_col = (uint32_t)(g * AL_BN), o_col = (uint32_t)(AL_O_COL + g * AL_HD);
        const int q_lo = g ? q_lo1 : q_lo0, pos_lo = start_pos + q_lo;
        const int pos = pos_lo + r, first = gb_first_key(pos, window), first_last = gb_first_key(pos_lo + AL_BM - 1, window);
        float m_run = AL_NEG_BIG, l_run = 0.f;
        bool ok = true;
        int stage = 0, phase = 0;                      // of the keys
        // A branch around the arrival for the first three quarters of P: across it the compiler forms no weights of the last quarter, which it
        // would do first otherwise (113 us of 109).
        auto gave_up = [&]() {
            if (!__any_sync(0xffffffffu, *abort_flag)) return false;
            ok = false;
            return true;
        };
        for (int j = 0; j < total; ++j) {
            const int key0 = (kt_begin + j) * AL_BN;
            if (!mbar_wait_warp(&sh.s_full[g][stage], phase, abort_flag, status)) { ok = false; break; }
            if (++stage == AL_KSTAGES) { stage = 0; phase ^= 1; }
            tc_fence_after();
            uint32_t sv[AL_BN];
            tmem_load128(lane_base + s_col, sv);
            if (key0 + AL_BN - 1 > pos_lo || key0 < first_last) {
#pragma unroll
                for (int k = 0; k < AL_BN; ++k)
                    if (key0 + k > pos || key0 + k < first) sv[k] = __float_as_uint(AL_NEG_BIG);
            }
            float mx4[4] = {AL_NEG_BIG, AL_NEG_BIG, AL_NEG_BIG, AL_NEG_BIG};
#pragma unroll
            for (int k = 0; k < AL_BN; k += 8)
#pragma unroll
                for (int u = 0; u < 4; ++u) mx4[u] = al_max3(mx4[u], __uint_as_float(sv[k + 2 * u]), __uint_as_float(sv[k + 2 * u + 1]));
            const float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3]));
            // the running maximum rises, and O_g is rescaled, only when it is exceeded by more than 2^8 in the exponent
            const bool raise = (mx - m_run) * sl2 > 8.0f;
            if (j == 0) {
                if (raise) m_run = mx;
            } else if (__any_sync(0xffffffffu, raise)) {
                // O += P V of the previous tile is complete (these scores were issued behind it)
                if (!mbar_wait_warp(&sh.pv_done[g][(j - 1) % AL_VSTAGES], ((j - 1) / AL_VSTAGES) & 1, abort_flag, status)) { ok = false; break; }
                tc_fence_after();
                const float corr = raise ? al_exp2((m_run - mx) * sl2) : 1.0f;
                if (raise) m_run = mx;
                l_run *= corr;
#pragma unroll
                for (int c = 0; c < AL_HD; c += 16) {
                    uint32_t ov[16];
                    tmem_load16(lane_base + o_col + (uint32_t)c, ov);
#pragma unroll
                    for (int k = 0; k < 16; ++k) ov[k] = __float_as_uint(__uint_as_float(ov[k]) * corr);
                    al_store16(lane_base + o_col + (uint32_t)c, ov);
                }
            }
            // P = exp2(S sl2 - m sl2). A masked key holds -1e30 and comes out as exactly 0; a row that has seen no key yet (its maximum is still
            // -1e30) must not cancel that, so its offset is 0.
            const float msl = m_run <= AL_NEG_BIG ? 0.f : m_run * sl2;
            const float2 scale2 = make_float2(sl2, sl2), off2 = make_float2(-msl, -msl);
            float2 l2[4] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f), make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
            for (int part = 0; part < AL_BN; part += 32) {
                uint32_t pw[16];
#pragma unroll
                for (int c = 0; c < 32; c += 2) {
                    const float2 y = __ffma2_rn(make_float2(__uint_as_float(sv[part + c]), __uint_as_float(sv[part + c + 1])), scale2, off2);
                    const float2 p = make_float2(al_exp2(y.x), al_exp2(y.y));
                    l2[(c >> 1) & 3] = __fadd2_rn(l2[(c >> 1) & 3], p);
                    pw[c >> 1] = pack2(__float_as_uint(p.x), __float_as_uint(p.y));
                }
                al_store16(lane_base + s_col + (uint32_t)(part / 2), pw);
                if (part == 64 && gave_up()) break;
                if (part >= 64) {      // three quarters, and the rest
                    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(part == 64 ? &sh.p_most[g] : &sh.p_ready[g]);
                    if (part == 64 && gave_up()) break;
                }
            }
            const float2 lsum = __fadd2_rn(__fadd2_rn(l2[0], l2[1]), __fadd2_rn(l2[2], l2[3]));
            l_run += lsum.x + lsum.y;
        }
        if (ok && total > 0) ok = mbar_wait_warp(&sh.pv_done[g][(total - 1) % AL_VSTAGES], ((total - 1) / AL_VSTAGES) & 1, abort_flag, status);
        if constexpr (CLUSTERS) {
            // O, maxima and sums to shared memory, where the cluster finds them: over the queries and keys, which both units have to be done with
            asm volatile("barrier.cta.sync 1, %0;" ::"r"(units * 128) : "memory");
            if (ok && total > 0) {
                tc_fence_after();
#pragma unroll
                for (int c = 0; c < AL_HD; c += 32) {
                    uint32_t ov[32];
                    tmem_load32(lane_base + o_col + (uint32_t)c, ov);
#pragma unroll
                    for (int k = 0; k < 32; k += 4)
                        *reinterpret_cast<uint4*>(al_smem + al_piece(g, r, (c + k) / 4)) = make_uint4(ov[k], ov[k + 1], ov[k + 2], ov[k + 3]);
                }
                float* stat = reinterpret_cast<float*>(al_smem + AL_STAT_OFF) + g * 2 * AL_BM;
                stat[r] = m_run;
                stat[AL_BM + r] = l_run;
            }
        } else if (ok) {
            // O / l, 32 channels at a time, to global memory
            tc_fence_after();
            const float inv = l_run != 0.f ? 1.0f / l_run : 0.f;
            __nv_bfloat16* dst = out + (size_t)(row0 + q_lo + r) * out_stride + (size_t)(kvh * group + (u0 + g) % group) * AL_HD;
#pragma unroll
            for (int c = 0; c < AL_HD; c += 32) {
                uint32_t ov[32];
                tmem_load32(lane_base + o_col + (uint32_t)c, ov);
                if (q_lo + r < nrows) {
#pragma unroll
                    for (int k = 0; k < 32; k += 8) {
                        uint4 w;
                        w.x = pack2(__float_as_uint(__uint_as_float(ov[k]) * inv), __float_as_uint(__uint_as_float(ov[k + 1]) * inv));
                        w.y = pack2(__float_as_uint(__uint_as_float(ov[k + 2]) * inv), __float_as_uint(__uint_as_float(ov[k + 3]) * inv));
                        w.z = pack2(__float_as_uint(__uint_as_float(ov[k + 4]) * inv), __float_as_uint(__uint_as_float(ov[k + 5]) * inv));
                        w.w = pack2(__float_as_uint(__uint_as_float(ov[k + 6]) * inv), __float_as_uint(__uint_as_float(ov[k + 7]) * inv));
                        *reinterpret_cast<uint4*>(dst + c + k) = w;
                    }
                }
            }
        }
    }

    // ------------------------------------------------------------------------------- the cluster's shares of the keys
    if constexpr (CLUSTERS) {
        tc_fence_before();
        al_cluster_sync();                       // (every block comes here: all waits before are bounded)
        const int g = (warp - 2) >> 2, r = (warp & 3) * 32 + lane, q_lo = g == 1 ? q_lo1 : q_lo0;
        if (warp >= 2 && warp < AL_WARPS - 1 && g < units && q_lo + r < nrows) {
            // each block adds up and writes its part of a row's channels
            const float sl2 = scale * 1.4426950408889634f;
            float most = AL_NEG_BIG, sum = 0.f, f[AL_MAX_CLUSTER];
            bool whole = true;
#pragma unroll
            for (int b = 0; b < AL_MAX_CLUSTER; ++b)
                if (b < cluster) {
                    whole = whole && __float_as_uint(al_peer(&sh.abort_flag, b)) == 0;
                    f[b] = share(b + 1) > share(b) ? al_peer(reinterpret_cast<float*>(al_smem + AL_STAT_OFF) + g * 2 * AL_BM + r, b) : AL_NEG_BIG;
                    most = fmaxf(most, f[b]);
                }
#pragma unroll
            for (int b = 0; b < AL_MAX_CLUSTER; ++b)
                if (b < cluster) {
                    f[b] = al_exp2((f[b] - most) * sl2);
                    if (share(b + 1) > share(b)) sum = fmaf(al_peer(reinterpret_cast<float*>(al_smem + AL_STAT_OFF) + g * 2 * AL_BM + AL_BM + r, b), f[b], sum);
                }
            const float inv = sum != 0.f ? 1.0f / sum : 0.f;
            const int width = AL_HD / cluster, c0 = rank * width;
            __nv_bfloat16* dst = out + (size_t)(row0 + q_lo + r) * out_stride + (size_t)(kvh * group + (u0 + g) % group) * AL_HD;
            for (int c = c0; c < c0 + width && whole; c += 8) {
                float o[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int b = 0; b < AL_MAX_CLUSTER; ++b)
                    if (b < cluster && share(b + 1) > share(b))
#pragma unroll
                        for (int k = 0; k < 8; k += 4) {
                            const float4 v = al_peer4(al_smem + al_piece(g, r, (c + k) / 4), b);
                            o[k] = fmaf(v.x, f[b], o[k]); o[k + 1] = fmaf(v.y, f[b], o[k + 1]);
                            o[k + 2] = fmaf(v.z, f[b], o[k + 2]); o[k + 3] = fmaf(v.w, f[b], o[k + 3]);
                        }
                uint4 w;
                w.x = pack2(__float_as_uint(o[0] * inv), __float_as_uint(o[1] * inv));
                w.y = pack2(__float_as_uint(o[2] * inv), __float_as_uint(o[3] * inv));
                w.z = pack2(__float_as_uint(o[4] * inv), __float_as_uint(o[5] * inv));
                w.w = pack2(__float_as_uint(o[6] * inv), __float_as_uint(o[7] * inv));
                *reinterpret_cast<uint4*>(dst + c) = w;
            }
        }
        al_cluster_sync();                       // (shared memory is read until here)
    }

    // ------------------------------------------------------------------------------- wind down
    tc_fence_before();
    __syncthreads();
    if (warp == 0) {
        if (lane == 0 && sh.abort_flag) {
            // copies that were issued but never consumed may still be in flight: wait for them (bounded)
            const long long t0 = clock64();
            while (sh.q_issued && !mbar_try_wait(&sh.q_full, 0) && clock64() - t0 < TC_WAIT_CYCLES) {}
            for (int what = 0; what < 2; ++what)
                for (int it = sh.consumed[what]; it < sh.issued[what]; ++it) {
                    uint64_t* bar = what == 0 ? &sh.k_full[it % AL_KSTAGES] : &sh.v_full[it % AL_VSTAGES];
                    const int phase = (what == 0 ? it / AL_KSTAGES : it / AL_VSTAGES) & 1;
                    const long long t1 = clock64();
                    while (!mbar_try_wait(bar, phase) && clock64() - t1 < TC_WAIT_CYCLES) {}
                }
        }
        __syncwarp();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(AL_TMEM_COLS) : "memory");
    }
}

GB_EXPORT int gb_attention_prefill_128_supported(int nh, int nkv, int hd, int page_size) {
    return nkv > 0 && nh % nkv == 0 && hd == AL_HD && page_size >= 8 && page_size <= AL_BN && (page_size & (page_size - 1)) == 0;
}

// Rows of each request are consecutive: request s owns rows seq_first_row[s] .. seq_first_row[s+1]-1, at positions seq_start_pos[s] + local index.
// q, out: bfloat16, rows aligned to 16 bytes; kcache, vcache: [num_pages, nkv, page_size, 128] contiguous.
GB_EXPORT int gb_attention_prefill_128(const void* q, long long q_stride, int n_rows, void* out, long long out_stride, const void* kcache,
                                       const void* vcache, const int* block_tables, int max_pages, const int* seq_first_row, const int* seq_start_pos,
                                       int num_seqs, int max_rows_per_seq, int max_context, int nh, int nkv, int hd, int page_size, long long num_pages, float scale,
                                       int window, int* status, cudaStream_t stream) {
    GB_REQUIRE(gb_attention_prefill_128_supported(nh, nkv, hd, page_size),
               "gb_attention_prefill_128: %d/%d heads of %d in pages of %d (a power of two, 8..128) are not built", nh, nkv, hd, page_size);
    GB_REQUIRE(q_stride % 8 == 0 && (uintptr_t)q % 16 == 0 && q_stride >= (long long)nh * hd && out_stride % 8 == 0 && (uintptr_t)out % 16 == 0,
               "gb_attention_prefill_128: rows must be 16-byte aligned");
    GB_REQUIRE((uintptr_t)kcache % 16 == 0 && (uintptr_t)vcache % 16 == 0, "gb_attention_prefill_128: the pages must be 16-byte aligned");
    GB_REQUIRE(num_seqs >= 0 && num_seqs <= 65535 && max_pages > 0 && status != nullptr && n_rows >= 0 && window >= 0,
               "gb_attention_prefill_128: bad batch shape");
    GB_REQUIRE(num_pages > 0 && num_pages * nkv * page_size < (1ll << 31) && (long long)max_pages * page_size < (1ll << 31) - 256,
               "gb_attention_prefill_128: the pages hold too many rows");
    if (num_seqs == 0 || n_rows == 0 || max_rows_per_seq <= 0) return 0;
    const long long pairs = ((long long)gb_ceil_div(max_rows_per_seq, AL_BM) * (nh / nkv) + 1) / 2;
    GB_REQUIRE(pairs <= 65535, "gb_attention_prefill_128: %d rows a request are too many for one launch", max_rows_per_seq);
    CUtensorMap mq, mk, mv;
    if (tc_make_map_2d(&mq, q, n_rows, (long long)nh * hd, q_stride, AL_BM, 64, "gb_attention_prefill_128")) return 1;
    if (tc_make_map_2d(&mk, kcache, num_pages * nkv * page_size, hd, hd, page_size, 64, "gb_attention_prefill_128")) return 1;
    if (tc_make_map_2d(&mv, vcache, num_pages * nkv * page_size, hd, hd, page_size, 64, "gb_attention_prefill_128")) return 1;
    // Few blocks behind many keys leave multiprocessors idle: clusters of two or four blocks then share a pair's keys, three tiles each at least. With
    // the unpacking, 32/8 heads, in clusters of 1 / 2 / 4: 256 rows behind 16,000 tokens 244 / 145 / 96 us, behind 4,000 73 / 53 / 46, 64 behind 2,000
    // 41 / 34 / 32, 16 behind 900 23 / 22 / 22; 4/2 heads, 512 behind 4,000 73 / 51 / 41. (Handing over and adding up costs some 8.)
    const long long blocks = pairs * nkv * num_seqs, reach = window > 0 && window + 2 * AL_BM < max_context ? window + 2 * AL_BM : max_context;
    int cluster = 1;
    while (cluster < AL_MAX_CLUSTER && blocks * cluster * 2 <= 148 && reach >= 3 * AL_BN * cluster * 2) cluster *= 2;
    const auto kernel = cluster > 1 ? attention_prefill_128_kernel<true> : attention_prefill_128_kernel<false>;
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, AL_SMEM);
    GB_REQUIRE(e == cudaSuccess, "gb_attention_prefill_128: %d bytes of shared memory refused: %s", AL_SMEM, cudaGetErrorString(e));
    int page_shift = 0;
    while ((1 << page_shift) < page_size) ++page_shift;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(nkv * cluster, num_seqs, (unsigned)pairs);
    cfg.blockDim = dim3(AL_WARPS * 32);
    cfg.dynamicSmemBytes = AL_SMEM;
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
    const cudaError_t launched = cudaLaunchKernelEx(&cfg, kernel, mq, mk, mv, (__nv_bfloat16*)out, out_stride, block_tables, max_pages,
                                                    seq_first_row, seq_start_pos, nh, nkv, page_size, page_shift, num_pages, scale, window, status);
    if (launched != cudaSuccess) {
        gb_set_error("gb_attention_prefill_128: launch failed: %s", cudaGetErrorString(launched));
        return 2;
    }
    return gb_check_launch("gb_attention_prefill_128");
}
