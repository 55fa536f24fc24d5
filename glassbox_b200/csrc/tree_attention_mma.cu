// Attention of trees of drafted tokens over the paged cache in bfloat16 on the tensor cores (mma.sync m16n8k16), head sizes 32, 64, 96 and 128.
//
// A block takes 16 WM query rows (rows of the tree x query heads that share the key/value head) of a request over its share of the keys, 64 at a time through a
// ring of stages: one thread's TMA copies of boxes of the page's keys x 64 channels in 128-byte-swizzled rows, for heads of 64 and 128; for 32
// and 96 every thread's 16-byte copies into rows padded by 16 bytes. WM x WK warps, each with 16 of the rows and 64 / WK of a stage's keys, so that small trees
// keep four warps at work. Softmax statistics and outputs are float32 (a maximum and a sum per row and warp, added up at the end); weights are rounded to bfloat16
// on their way into the second product, 2^-9 of each.
//
// Masks are looked at only where a warp's keys hold some that a row may not see: bits of the tree come as 32 at a time. There a value that is not a finite
// number must not meet a weight of zero, so such values are zero in the product and go to the rows that see them one by one.
//
// What bounds it: keys and values are read once, 256 bytes of them for a row's 128 products and an exponential. 16 trees of 32 rows, 32/32 heads of 64, behind
// 4,095 tokens (541 MB): 129 us, 4.2 TB/s; there a warp's chain of scores, softmax and product, of which a multiprocessor has 16 under way (1.9 instructions a cycle, tensor
// cores 28 % busy), and about 7 us of a start and an end beside each item. Where items are few, that and a tile's trip: 1 tree of 8 rows, 9/3 heads of 64, behind 1,023 tokens 10 us.
#include "tcgen05.cuh"
#include "tree_attention.cuh"

#include <cooperative_groups.h>
#include <type_traits>

constexpr int TM_KEYS = 64, TM_MAX_PAGES = 1024, TM_MAX_CLUSTER = 8;

__device__ __forceinline__ void tm_copy16(uint32_t to, const void* from, bool valid) {
    const int bytes = valid ? 16 : 0;
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(bytes) : "memory");
}
__device__ __forceinline__ void tm_ldmatrix(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void tm_ldmatrix_t(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void tm_mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float tm_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t tm_pack(float lo, float hi) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}
// Two values, those that are not finite numbers as zero.
__device__ __forceinline__ uint32_t tm_finite(uint32_t two) {
    if ((two & 0x7f80u) == 0x7f80u) two &= 0xffff0000u;
    if ((two & 0x7f800000u) == 0x7f800000u) two &= 0xffffu;
    return two;
}

template <int HD, int WM, int WK, bool CLUSTER>
struct TmShape {
    static constexpr bool TMA = HD % 64 == 0;      // blocks of 64 channels in 128-byte-swizzled rows, else padded rows that threads copy
    // (an even cut of 16 trees of 32 rows, 32/32 heads of 64, 4,095 tokens: four blocks a multiprocessor of three stages 129 us, three of four 143; clusters of 8 trees
    // of 16 rows, 15/5 heads of 64, 2,500 tokens: 18 and 16.5)
    static constexpr int STAGES = HD == 64 && CLUSTER ? 4 : 3, BLOCKS = WM * WK == 8 ? (HD > 64 ? 1 : 2) : HD > 64 ? 2 : HD == 64 && CLUSTER ? 3 : 4;
    static constexpr int COLS = HD / 64, BLOCK = TM_KEYS * 128;
    static constexpr int PITCH = TMA ? 128 : HD * 2 + 16, TILE = TMA ? COLS * BLOCK : TM_KEYS * PITCH, THREADS = WM * WK * 32, ROWS = WM * 16, KW = TM_KEYS / WK, P = HD + 2;
    static constexpr int SMEM = 2 * STAGES * TILE + TM_MAX_PAGES * 4;
    static_assert(WM * WK * 16 * P * 4 <= 2 * STAGES * TILE, "the warps' results lie over the stages");
};

// CLUSTER: the blocks of a cluster share one item's keys (blockIdx.x of gridDim.x of them; item: blockIdx.y, request: blockIdx.z) and add up through distributed
// shared memory. Otherwise all items' tiles of keys are cut evenly among the blocks; what a block finds of an item that it shares with others goes to the
// scratch, piece number (item + block), and tree_pieces_kernel adds up.
template <int HD, int WM, int WK, bool CLUSTER>
__global__ void __launch_bounds__(WM* WK * 32, TmShape<HD, WM, WK, CLUSTER>::BLOCKS) tree_attention_mma_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                                                                         const TreeArgs a, int num_seqs) {
    namespace cg = cooperative_groups;
    using Sh = TmShape<HD, WM, WK, CLUSTER>;
    constexpr bool TMA = Sh::TMA;
    constexpr int STAGES = Sh::STAGES, NW = WM * WK;
    // Tiles that are under way beside the one worked on: with TMA one stage less than there are, so that a warp may be a tile behind the one that asks for the
    // next.
    constexpr int AHEAD = TMA ? STAGES - 2 : STAGES - 1;
    constexpr int CH = HD / 8, KS = HD / 16, NT = HD / 8, KW = Sh::KW, KT = KW / 8, P = Sh::P;
    extern __shared__ __align__(1024) unsigned char tm_mem[];
    __shared__ __align__(8) uint64_t full[STAGES], done[STAGES];      // TMA -> the warps: a stage's keys and values are there; the warps -> warp 0: they are read
    __shared__ int abort_word;
    volatile int* abort_flag = &abort_word;
    unsigned char* Ks = tm_mem;
    unsigned char* Vs = tm_mem + STAGES * Sh::TILE;
    int* pages = reinterpret_cast<int*>(tm_mem + 2 * STAGES * Sh::TILE);
    float* res = reinterpret_cast<float*>(tm_mem);           // the warps' results: [WK][ROWS][channels, maximum, sum]
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, wm = warp % WM, wk = warp / WM, g = lane >> 2, t = lane & 3;
    const int G = a.nh / a.nkv;
    gb_pdl_launch_dependents();
    gb_pdl_wait();
    __nv_bfloat16* out = (__nv_bfloat16*)a.out;
    const __nv_bfloat16* kc = (const __nv_bfloat16*)a.kcache;
    const __nv_bfloat16* vc = (const __nv_bfloat16*)a.vcache;
    const float sl2 = a.scale * 1.4426950408889634f;
    int shift = 0;
    while ((1 << shift) < a.page_size) ++shift;
    int loaded = 0;                                           // tiles that the block has taken from its stages
    if constexpr (TMA) {
        if (smem_u32(tm_mem) & 1023u) {                       // swizzled tiles want 1024-byte alignment: refuse rather than compute nonsense
            if (tid == 0) atomicOr(a.status, GB_STATUS_WAIT_TIMEOUT);
            return;
        }
        if (tid == 0) {
            for (int i = 0; i < STAGES; ++i) { mbar_init(&full[i], 1); mbar_init(&done[i], NW); }
            abort_word = 0;
            asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        }
    }

    // One item's tiles [tile0, tile1) of keys (from the first that any row sees); `tiles` it has in all; `piece`: where a part of them goes.
    auto work = [&](const TreeSeq& s, int kvh, int m0, int tile0, int tile1, int tiles_all, long long piece) {
        const int M = s.rows * G;
        // the thread's two rows: g and g + 8 of the warp's
        int row[2], head[2], pos[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int m = m0 + wm * 16 + g + 8 * h;
            row[h] = m < M ? s.row0 + m / G : -1;
            head[h] = kvh * G + m % G;
        }
        const int base = s.key_lo / TM_KEYS * TM_KEYS, k_begin = base + tile0 * TM_KEYS, k_end = min(s.length, base + tile1 * TM_KEYS), tiles = tile1 - tile0;
        const int page_lo = k_begin >> shift, n_pages = tiles > 0 ? ((k_end - 1) >> shift) - page_lo + 1 : 0;
        const bool staged = n_pages <= TM_MAX_PAGES;
        bool bad = false;
        // (loads whose results are not used at once come first: a warp waits where it needs one)
        uint32_t qf[KS][4];
#pragma unroll
        for (int k = 0; k < KS; ++k)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int h = i & 1;
                qf[k][i] = row[h] >= 0 ? *reinterpret_cast<const uint32_t*>((const __nv_bfloat16*)a.q + (size_t)row[h] * a.q_stride + head[h] * HD + 16 * k + 8 * (i >> 1) + 2 * t) : 0u;
            }
        unsigned word[2];                             // of the rows' bits, where there is one
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            pos[h] = row[h] >= 0 ? a.positions[row[h]] : -1;
            word[h] = row[h] >= 0 && a.words == 1 ? (unsigned)a.visible[row[h]] : 0u;
        }
        // (what the block did before is done with shared memory, and what it wrote over the stages lies before the copies to come)
        if constexpr (TMA) asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncthreads();
        if (staged)
            for (int i = tid; i < n_pages; i += Sh::THREADS) pages[i] = s.page(a, page_lo + i);
        __syncthreads();
        auto load = [&](int tile) {
            const int k0 = k_begin + tile * TM_KEYS, stage = (loaded + tile) % STAGES;
            if constexpr (TMA) {
                // A lane a box of 64 channels of a page's keys. What no row sees, or is missing, lies behind all pages, where a copy reads zeros; keys behind the
                // request's last in its page are masked.
                if (warp != 0) return;
                const int box = min(a.page_size, TM_KEYS), count = TM_KEYS / box, which = lane & 1, col = lane >> 1 & (Sh::COLS - 1), i = lane / (2 * Sh::COLS);
                const int use = (loaded + tile) / STAGES;      // of the stage
                if (use > 0) mbar_wait(&done[stage], (use - 1) & 1, abort_flag, a.status);
                if (__any_sync(0xffffffffu, *abort_flag)) return;
                if (lane == 0) mbar_expect_tx(&full[stage], 2 * Sh::TILE);
                __syncwarp();
                for (int j = i; j < count; j += 16 / Sh::COLS) {
                    const int key = k0 + j * box;
                    int at = (int)(a.num_pages * a.nkv * a.page_size);
                    if (key < k_end && key + box > s.key_lo) {
                        const int page = staged ? pages[(key >> shift) - page_lo] : s.page(a, key >> shift);
                        if (page >= 0) at = (page * a.nkv + kvh) * a.page_size + (key & (a.page_size - 1));
                        else bad = true;
                    }
                    tma_load_2d((which ? Vs : Ks) + stage * Sh::TILE + col * Sh::BLOCK + j * box * 128, which ? &map_v : &map_k, &full[stage], col * 64, at);
                }
                return;
            }
            const uint32_t kb = smem_u32(Ks + stage * Sh::TILE), vb = smem_u32(Vs + stage * Sh::TILE);
#pragma unroll
            for (int i = 0; i < TM_KEYS * CH / Sh::THREADS; ++i) {
                const int idx = tid + i * Sh::THREADS, r = idx / CH, c = idx % CH, key = k0 + r;
                int page = -1;
                if (key >= s.key_lo && key < k_end) {
                    page = staged ? pages[(key >> shift) - page_lo] : s.page(a, key >> shift);
                    if (page < 0) bad = true;
                }
                const size_t at = page < 0 ? 0 : (((size_t)page * a.nkv + kvh) * a.page_size + (key & (a.page_size - 1))) * HD + c * 8;
                tm_copy16(kb + r * Sh::PITCH + c * 16, kc + at, page >= 0);
                tm_copy16(vb + r * Sh::PITCH + c * 16, vc + at, page >= 0);
            }
        };
        // 16 bytes of a lane's row of a tile for ldmatrix: keys' rows by (lane >> 4) and lane & 7, values' by (lane >> 3) & 1 and lane & 7; pieces in pairs
        const int k_half = lane >> 3 & 1, v_half = lane >> 4, turn = lane & 7;
        auto piece_at = [&](int pair, int half) -> uint32_t {
            if constexpr (TMA) return (uint32_t)(pair / 4 * Sh::BLOCK + (((pair % 4 * 2 + half) ^ turn) << 4));
            return (uint32_t)(pair * 32 + half * 16);
        };
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            if (i < tiles) load(i);
            if constexpr (!TMA) asm volatile("cp.async.commit_group;" ::: "memory");
        }
        float m_run[2] = {-INFINITY, -INFINITY}, l_run[2] = {0.f, 0.f}, acc[NT][4];
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[j][e] = 0.f;
        for (int tile = 0; tile < tiles; ++tile) {
            // the tile is there, and the one before has been read
            const int stage = (loaded + tile) % STAGES;
            if constexpr (!TMA) {
                asm volatile("cp.async.wait_group %0;" ::"n"(AHEAD - 1) : "memory");
                __syncthreads();
            }
            if (tile + AHEAD < tiles) load(tile + AHEAD);
            if constexpr (!TMA) asm volatile("cp.async.commit_group;" ::: "memory");
            if constexpr (TMA) mbar_wait(&full[stage], (loaded + tile) / STAGES & 1, abort_flag, a.status);      // (one that runs out is reported)
            const int k0 = k_begin + tile * TM_KEYS + wk * KW;      // of the warp's keys
            const unsigned char* vs = Vs + stage * Sh::TILE + wk * KW * Sh::PITCH;
            const uint32_t kb = smem_u32(Ks + stage * Sh::TILE) + (wk * KW + v_half * 8 + turn) * Sh::PITCH, vb = smem_u32(vs) + (k_half * 8 + turn) * Sh::PITCH;
            float sc[KT][4];
#pragma unroll
            for (int j = 0; j < KT; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) sc[j][e] = 0.f;
#pragma unroll
            for (int j = 0; j < KT; j += 2)
#pragma unroll
                for (int k = 0; k < KS; ++k) {
                    uint32_t b[4];
                    tm_ldmatrix(b, kb + j * 8 * Sh::PITCH + piece_at(k, k_half));
                    tm_mma(sc[j], qf[k], b[0], b[1]);
                    tm_mma(sc[j + 1], qf[k], b[2], b[3]);
                }
            bool masked = k0 + KW > s.start;
            if (a.window > 0) masked = masked || __any_sync(0xffffffffu, max(pos[0], pos[1]) - k0 >= a.window);
            bool odd = false;                             // a value here is not a finite number
            if (masked) {
                unsigned see[2][(KW + 31) / 32];
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int w = 0; w < (KW + 31) / 32; ++w) see[h][w] = tree_bits(a, s.rows, row[h], k0 + 32 * w - s.start, word[h]);
#pragma unroll
                for (int j = 0; j < KT; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int i = 8 * j + 2 * t + (e & 1), key = k0 + i;
                        bool ok = see[e >> 1][i >> 5] >> (i & 31) & 1u;
                        if (a.window > 0 && ok) ok = pos[e >> 1] - (key < s.start ? key : a.positions[s.row0 + key - s.start]) < a.window;
                        if (!ok) sc[j][e] = -INFINITY;
                    }
                for (int i = lane; i < KW * CH; i += 32) {
                    const int key = i / CH, c = i % CH;
                    const uint4 v = *reinterpret_cast<const uint4*>(vs + key * Sh::PITCH + (TMA ? c / 8 * Sh::BLOCK + ((c % 8) ^ (key & 7)) * 16 : c * 16));
                    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                    for (int e = 0; e < 4; ++e) odd = odd || (w[e] & 0x7f80u) == 0x7f80u || (w[e] & 0x7f800000u) == 0x7f800000u;
                }
                odd = __any_sync(0xffffffffu, odd);
            }
            float mx[2] = {-INFINITY, -INFINITY}, off[2], corr[2];
#pragma unroll
            for (int j = 0; j < KT; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    // (masked ones stay minus infinity at any scale, also a negative one)
                    sc[j][e] = masked && sc[j][e] == -INFINITY ? -INFINITY : sc[j][e] * sl2;
                    mx[e >> 1] = fmaxf(mx[e >> 1], sc[j][e]);
                }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 1));
                mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 2));
                const float m_new = fmaxf(m_run[h], mx[h]);
                off[h] = m_new == -INFINITY ? 0.f : m_new;
                corr[h] = tm_exp2(m_run[h] - off[h]);
                m_run[h] = m_new;
                l_run[h] *= corr[h];
            }
#pragma unroll
            for (int j = 0; j < KT; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    sc[j][e] = tm_exp2(sc[j][e] - off[e >> 1]);
                    l_run[e >> 1] += sc[j][e];            // (this thread's share)
                }
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[j][e] *= corr[e >> 1];
            auto product = [&](auto some_odd) {
#pragma unroll
                for (int b = 0; b < KW / 16; ++b) {
                    const uint32_t p[4] = {tm_pack(sc[2 * b][0], sc[2 * b][1]), tm_pack(sc[2 * b][2], sc[2 * b][3]), tm_pack(sc[2 * b + 1][0], sc[2 * b + 1][1]),
                                           tm_pack(sc[2 * b + 1][2], sc[2 * b + 1][3])};
#pragma unroll
                    for (int j = 0; j < NT; j += 2) {
                        uint32_t v[4];
                        tm_ldmatrix_t(v, vb + b * 16 * Sh::PITCH + piece_at(j / 2, v_half));
                        if constexpr (decltype(some_odd)::value) {
#pragma unroll
                            for (int e = 0; e < 4; ++e) v[e] = tm_finite(v[e]);
                        }
                        tm_mma(acc[j], p, v[0], v[1]);
                        tm_mma(acc[j + 1], p, v[2], v[3]);
                    }
                }
            };
            if (!odd) {
                product(std::false_type());
            } else {
                product(std::true_type());
#pragma unroll
                for (int j = 0; j < KT; ++j)
#pragma unroll
                    for (int e = 0; e < 2; ++e)
                        for (int tt = 0; tt < 4; ++tt) {
                            const float p0 = __shfl_sync(0xffffffffu, sc[j][e], (lane & ~3) | tt), p1 = __shfl_sync(0xffffffffu, sc[j][2 + e], (lane & ~3) | tt);
                            const int key = 8 * j + 2 * tt + e;
                            const unsigned char* v = vs + key * Sh::PITCH + 4 * t;
#pragma unroll
                            for (int c = 0; c < NT; ++c) {
                                const uint32_t two = *reinterpret_cast<const uint32_t*>(v + (TMA ? c / 8 * Sh::BLOCK + ((c % 8) ^ (key & 7)) * 16 : c * 16));
                                const float lo = __uint_as_float(two << 16), hi = __uint_as_float(two & 0xffff0000u);
                                const bool odd_lo = (two & 0x7f80u) == 0x7f80u, odd_hi = (two & 0x7f800000u) == 0x7f800000u;
                                if (p0 != 0.f && odd_lo) acc[c][0] += p0 * lo;
                                if (p0 != 0.f && odd_hi) acc[c][1] += p0 * hi;
                                if (p1 != 0.f && odd_lo) acc[c][2] += p1 * lo;
                                if (p1 != 0.f && odd_hi) acc[c][3] += p1 * hi;
                            }
                        }
            }
            if constexpr (TMA) {
                __syncwarp();
                if (lane == 0) mbar_arrive(&done[stage]);
            }
        }
        if constexpr (!TMA) asm volatile("cp.async.wait_group 0;" ::: "memory");
        if constexpr (TMA)
            if (*abort_flag && tid == 0)                  // copies that were issued and not waited for to the end may still be in flight: once more, bounded
                for (int tile = max(0, tiles - STAGES); tile < tiles; ++tile) {
                    const long long t0 = clock64();
                    while (!mbar_try_wait(&full[(loaded + tile) % STAGES], (loaded + tile) / STAGES & 1) && clock64() - t0 < TC_WAIT_CYCLES) {}
                }
        loaded += tiles;
        if (bad) atomicOr(a.status, GB_STATUS_BAD_SLOT);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            l_run[h] += __shfl_xor_sync(0xffffffffu, l_run[h], 1);
            l_run[h] += __shfl_xor_sync(0xffffffffu, l_run[h], 2);
        }
        __syncthreads();                              // (all stages have been read)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            float* to = res + ((size_t)(wk * WM + wm) * 16 + g + 8 * h) * P;
#pragma unroll
            for (int j = 0; j < NT; ++j) *reinterpret_cast<float2*>(to + 8 * j + 2 * t) = make_float2(acc[j][2 * h], acc[j][2 * h + 1]);
            if (t == 0) *reinterpret_cast<float2*>(to + HD) = make_float2(m_run[h], l_run[h]);
        }
        const int parts = CLUSTER ? gridDim.x : 1, rank = CLUSTER ? blockIdx.x : 0;
        if (CLUSTER && parts > 1) cg::this_cluster().sync(); else __syncthreads();
        // A pair of channels of every parts-th row; all loads of other blocks' results come first: one trip.
        auto add_up = [&](auto blocks) {
            constexpr int MOST = decltype(blocks)::value;
            constexpr int E = MOST * WK <= 2 ? 4 : MOST * WK <= 8 ? 2 : 1, LANES = HD / 2 / E;      // pairs of a thread, LANES pairs apart: as many as its registers hold
            for (int i = tid; i < (Sh::ROWS - rank + MOST - 1) / MOST * LANES; i += Sh::THREADS) {
                const int r = i / LANES * MOST + rank, c = i % LANES * 2, m = m0 + r;
                if (m >= M) break;
                float2 ml[MOST][WK], v[MOST][WK][E];
#pragma unroll
                for (int b = 0; b < MOST; ++b) {
                    const float* all = MOST > 1 ? cg::this_cluster().map_shared_rank(res, b) : res;
#pragma unroll
                    for (int w = 0; w < WK; ++w) {
                        const float* from = all + ((size_t)w * Sh::ROWS + r) * P;
                        ml[b][w] = *reinterpret_cast<const float2*>(from + HD);
#pragma unroll
                        for (int e = 0; e < E; ++e) v[b][w][e] = *reinterpret_cast<const float2*>(from + c + 2 * LANES * e);
                    }
                }
                float top = -INFINITY, l = 0.f, x[E], y[E];
#pragma unroll
                for (int e = 0; e < E; ++e) x[e] = y[e] = 0.f;
#pragma unroll
                for (int b = 0; b < MOST; ++b)
#pragma unroll
                    for (int w = 0; w < WK; ++w) top = fmaxf(top, ml[b][w].x);
                const float o = top == -INFINITY ? 0.f : top;
#pragma unroll
                for (int b = 0; b < MOST; ++b)
#pragma unroll
                    for (int w = 0; w < WK; ++w) {
                        const float f = tm_exp2(ml[b][w].x - o);
                        l = fmaf(ml[b][w].y, f, l);
#pragma unroll
                        for (int e = 0; e < E; ++e) {
                            x[e] = fmaf(v[b][w][e].x, f, x[e]);
                            y[e] = fmaf(v[b][w][e].y, f, y[e]);
                        }
                    }
                if (CLUSTER || tile1 - tile0 == tiles_all) {
                    const float inv = l != 0.f ? 1.0f / l : 0.f;
                    __nv_bfloat16* to = out + (size_t)(s.row0 + m / G) * a.out_stride + (kvh * G + m % G) * HD + c;
#pragma unroll
                    for (int e = 0; e < E; ++e) *reinterpret_cast<uint32_t*>(to + 2 * LANES * e) = tm_pack(x[e] * inv, y[e] * inv);
                } else {
                    float* part = a.parts + ((size_t)piece * Sh::ROWS + r) * P;
#pragma unroll
                    for (int e = 0; e < E; ++e) *reinterpret_cast<float2*>(part + c + 2 * LANES * e) = make_float2(x[e], y[e]);
                    if (c == 0) *reinterpret_cast<float2*>(part + HD) = make_float2(top, l);
                }
            }
        };
        if (!CLUSTER || parts == 1) add_up(std::integral_constant<int, 1>());
        else if (parts == 2) add_up(std::integral_constant<int, 2>());
        else if (parts == 4) add_up(std::integral_constant<int, 4>());
        else add_up(std::integral_constant<int, TM_MAX_CLUSTER>());
        if (CLUSTER && parts > 1) cg::this_cluster().sync();      // (shared memory is read until here)
    };
    auto zeros = [&](const TreeSeq& s) {              // a padding request's rows
        for (int i = tid; i < s.rows * a.nh * (HD / 2); i += Sh::THREADS)
            *reinterpret_cast<uint32_t*>(out + (size_t)(s.row0 + i / (a.nh * (HD / 2))) * a.out_stride + i % (a.nh * (HD / 2)) * 2) = 0u;
    };

    if constexpr (CLUSTER) {
        const TreeSeq s(a, blockIdx.z);
        const int m0 = blockIdx.y / a.nkv * Sh::ROWS;
        if (s.start < 0 || m0 >= s.rows * G) {        // (the same for the whole cluster)
            if (s.start < 0 && blockIdx.x == 0 && blockIdx.y == 0) zeros(s);
            return;
        }
        const int all = s.tiles(TM_KEYS), share = (all + gridDim.x - 1) / gridDim.x, tile0 = min(all, (int)blockIdx.x * share);
        work(s, blockIdx.y % a.nkv, m0, tile0, min(all, tile0 + share), all, 0);
    } else {
        TreeCut cut(a, num_seqs, Sh::ROWS, TM_KEYS, gridDim.x, TREE_LEAST_SHARE);
        long long at = min(cut.total, blockIdx.x * cut.share);
        const long long end = min(cut.total, at + cut.share);
        if (at < end) {
            cut.seek(at);
            while (at < end) {
                const TreeSeq s(a, cut.seq);
                const int all = s.tiles(TM_KEYS), m_tiles = (s.rows * G + Sh::ROWS - 1) / Sh::ROWS;
                const long long off = at - cut.tile0;
                const int item = (int)(off / all), tile0 = (int)(off % all), tile1 = (int)min((long long)all, tile0 + (end - at));
                work(s, item / m_tiles, item % m_tiles * Sh::ROWS, tile0, tile1, all, cut.item0 + item + blockIdx.x);
                at += tile1 - tile0;
                if (at < end) cut.reach(at);
            }
        }
        for (int seq = blockIdx.x; seq < num_seqs; seq += gridDim.x) {
            if (a.start_pos[seq] >= 0) continue;
            const TreeSeq s(a, seq);
            zeros(s);
        }
    }
}

// Adds up the pieces of items that several blocks share: 8 rows of an item a block (x: piece of rows and item, y: request).
template <int HD, int ROWS>
__global__ void __launch_bounds__(128) tree_pieces_kernel(const TreeArgs a, int num_seqs, int m_tiles_most, int blocks) {
    constexpr int P = HD + 2, EACH = 8;
    gb_pdl_launch_dependents();
    gb_pdl_wait();
    TreeCut cut(a, num_seqs, ROWS, TM_KEYS, blocks, TREE_LEAST_SHARE);
    const int seq = blockIdx.y, G = a.nh / a.nkv, row_part = blockIdx.x % (ROWS / EACH), rest = blockIdx.x / (ROWS / EACH);
    const int m_tile = rest % m_tiles_most, kvh = rest / m_tiles_most;
    const TreeSeq s(a, seq);
    const int m_tiles = (s.rows * G + ROWS - 1) / ROWS, m0 = m_tile * ROWS + row_part * EACH, M = s.rows * G;
    if (s.start < 0 || m0 >= M) return;
    cut.seek_seq(seq);
    const int all = s.tiles(TM_KEYS), item = kvh * m_tiles + m_tile;
    const long long t0 = cut.tile0 + (long long)item * all, b0 = t0 / cut.share, b1 = (t0 + all - 1) / cut.share;
    if (b0 == b1) return;
    const float* pieces = a.parts + (size_t)(cut.item0 + item) * ROWS * P + (size_t)(row_part * EACH) * P;
    for (int i = threadIdx.x; i < EACH * (HD / 2); i += 128) {
        const int r = i / (HD / 2), c = i % (HD / 2) * 2, m = m0 + r;
        if (m >= M) break;
        const float* mine = pieces + r * P;
        float top = -INFINITY, l = 0.f, x = 0.f, y = 0.f;
#pragma unroll 4
        for (long long b = b0; b <= b1; ++b) top = fmaxf(top, mine[b * ROWS * P + HD]);
        const float o = top == -INFINITY ? 0.f : top;
#pragma unroll 4
        for (long long b = b0; b <= b1; ++b) {
            const float* from = mine + b * ROWS * P;
            const float2 ml = *reinterpret_cast<const float2*>(from + HD), v = *reinterpret_cast<const float2*>(from + c);
            const float f = tm_exp2(ml.x - o);
            l = fmaf(ml.y, f, l);
            x = fmaf(v.x, f, x);
            y = fmaf(v.y, f, y);
        }
        const float inv = l != 0.f ? 1.0f / l : 0.f;
        *reinterpret_cast<uint32_t*>((__nv_bfloat16*)a.out + (size_t)(s.row0 + m / G) * a.out_stride + (kvh * G + m % G) * HD + c) = tm_pack(x * inv, y * inv);
    }
}

template <int HD, int WM, int WK>
static int tm_launch(const TreeArgs& a, const TreePlan& plan, int num_seqs, int max_rows, cudaStream_t stream) {
    using Sh = TmShape<HD, WM, WK, true>;             // (what both forms share)
    CUtensorMap mk = {}, mv = {};
    if constexpr (Sh::TMA) {
        const int box = a.page_size < TM_KEYS ? a.page_size : TM_KEYS;
        if (tc_make_map_2d(&mk, a.kcache, a.num_pages * a.nkv * a.page_size, HD, HD, box, 64, "gb_tree_attention")) return 1;
        if (tc_make_map_2d(&mv, a.vcache, a.num_pages * a.nkv * a.page_size, HD, HD, box, 64, "gb_tree_attention")) return 1;
    }
    const int m_tiles = gb_ceil_div((long long)max_rows * (a.nh / a.nkv), Sh::ROWS);
    GB_REQUIRE((long long)m_tiles * a.nkv * (Sh::ROWS / 8) <= 65535ll * 1024 && (long long)m_tiles * a.nkv <= 65535, "gb_tree_attention: %d rows a request are too many for one launch", max_rows);
    cudaError_t e;
    if (plan.cluster) {
        const auto kernel = tree_attention_mma_kernel<HD, WM, WK, true>;
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Sh::SMEM);
        GB_REQUIRE(e == cudaSuccess, "gb_tree_attention: %d bytes of shared memory refused: %s", Sh::SMEM, cudaGetErrorString(e));
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(plan.cluster, m_tiles * a.nkv, num_seqs);
        cfg.blockDim = dim3(Sh::THREADS);
        cfg.dynamicSmemBytes = Sh::SMEM;
        cfg.stream = stream;
        cudaLaunchAttribute attr[2];
        int na = 0;
        if (gb_pdl_enabled() & GB_PDL_ATTENTION) {
            attr[na].id = cudaLaunchAttributeProgrammaticStreamSerialization;
            attr[na].val.programmaticStreamSerializationAllowed = 1;
            ++na;
        }
        attr[na].id = cudaLaunchAttributeClusterDimension;
        attr[na].val.clusterDim.x = plan.cluster;
        attr[na].val.clusterDim.y = attr[na].val.clusterDim.z = 1;
        ++na;
        cfg.attrs = attr;
        cfg.numAttrs = na;
        e = cudaLaunchKernelEx(&cfg, kernel, mk, mv, a, num_seqs);
        GB_REQUIRE(e == cudaSuccess, "gb_tree_attention: launch failed: %s", cudaGetErrorString(e));
        return gb_check_launch("gb_tree_attention");
    }
    const auto kernel = tree_attention_mma_kernel<HD, WM, WK, false>;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, TmShape<HD, WM, WK, false>::SMEM);
    GB_REQUIRE(e == cudaSuccess, "gb_tree_attention: %d bytes of shared memory refused: %s", TmShape<HD, WM, WK, false>::SMEM, cudaGetErrorString(e));
    e = gb_launch(GB_PDL_ATTENTION, kernel, dim3(plan.blocks), dim3(Sh::THREADS), TmShape<HD, WM, WK, false>::SMEM, stream, mk, mv, a, num_seqs);
    GB_REQUIRE(e == cudaSuccess, "gb_tree_attention: launch failed: %s", cudaGetErrorString(e));
    e = gb_launch(GB_PDL_ATTENTION, tree_pieces_kernel<HD, Sh::ROWS>, dim3(m_tiles * a.nkv * (Sh::ROWS / 8), num_seqs), dim3(128), 0, stream, a, num_seqs, m_tiles, plan.blocks);
    GB_REQUIRE(e == cudaSuccess, "gb_tree_attention: launch failed: %s", cudaGetErrorString(e));
    return gb_check_launch("gb_tree_attention");
}

template <int HD>
static int tm_dispatch(const TreeArgs& a, const TreePlan& plan, int num_seqs, int max_rows, cudaStream_t stream) {
    switch (plan.rows) {
        case 16: return tm_launch<HD, 1, 4>(a, plan, num_seqs, max_rows, stream);
        case 32: return tm_launch<HD, 2, 2>(a, plan, num_seqs, max_rows, stream);
        case 64: return tm_launch<HD, 4, 1>(a, plan, num_seqs, max_rows, stream);
        default: return tm_launch<HD, 8, 1>(a, plan, num_seqs, max_rows, stream);
    }
}

int gb_tree_attention_mma(const TreeArgs& a, const TreePlan& plan, int num_seqs, int max_rows, cudaStream_t stream) {
    GB_REQUIRE(a.page_size >= 8 && (a.page_size & (a.page_size - 1)) == 0, "gb_tree_attention: pages of %d tokens (a power of two from 8 on) are not built here", a.page_size);
    GB_REQUIRE(a.num_pages * a.nkv * a.page_size < (1ll << 31), "gb_tree_attention: the pages hold too many rows");
    GB_REQUIRE((uintptr_t)a.kcache % 16 == 0 && (uintptr_t)a.vcache % 16 == 0 && (uintptr_t)a.q % 4 == 0 && a.q_stride % 2 == 0 && (uintptr_t)a.out % 4 == 0 && a.out_stride % 2 == 0,
               "gb_tree_attention: rows must be 4-byte aligned, pages 16-byte aligned");
    if (a.hd == 32) return tm_dispatch<32>(a, plan, num_seqs, max_rows, stream);
    if (a.hd == 64) return tm_dispatch<64>(a, plan, num_seqs, max_rows, stream);
    if (a.hd == 96) return tm_dispatch<96>(a, plan, num_seqs, max_rows, stream);
    GB_REQUIRE(a.hd == 128, "gb_tree_attention: heads of %d are not built here", a.hd);
    return tm_dispatch<128>(a, plan, num_seqs, max_rows, stream);
}

// More than 32 rows, and either many keys in all (of every request and key/value head, times the groups of 64 rows that read them here) or long ones: the kernel
// on tcgen05 has about 20 us of its own, and less for each key. Measured, this one and that (us): 16 trees of 24 rows, 32/8 heads of 128, behind 250 tokens 33 and
// 33, 600 41 and 23, 2,400 107 and 57; one of them behind 2,400 23 and 29, 4,800 35 and 31, 9,600 70 and 35; one of 64 rows behind 600 25 and 39, 2,400 57 and 33;
// 16 trees of 64 rows, 9/3 heads of 64, behind 600 31 and 31, 1,200 43 and 31; 4 of 40 rows, 32/32 heads of 128, behind 600 29 and 21, 2,400 66 and 51.
// With fewer query rows half of that kernel's work is on empty ones, and memory feeds either; it is ahead with long keys of few requests and heads, which clusters
// of eight blocks leave part of the GPU without (8 rows, 15/5 heads of 64, behind 4,095 tokens 16 and 23, 16,000 41 and 26, 64,000 74 and 39; 4 requests behind
// 16,000 45 and 33; 32/32 heads 45 and 47), and with 17 rows or more of 128 channels, whose products bound this kernel (32 rows, 32/8 heads, 4 requests behind
// 4,095 27 and 33, 16,000 69 and 65, 64,000 236 and 185; 16 rows 201 and 185).
static bool tree_takes_tc(int num_seqs, long long M, int nkv, int hd, int max_context) {
    const double keys = (double)max_context * num_seqs * nkv;
    if (M > 32) return (long long)max_context * gb_ceil_div(M, 128) >= 4096 || keys * gb_ceil_div(M, 64) >= 112 * 1024;
    return (max_context >= 8192 && num_seqs * nkv <= 24) || (hd == 128 && M > 16 && keys >= 512 * 1024);
}

// Clusters while every item's blocks find room at once, or all tiles evenly among the blocks that do and a second launch that adds up: whichever this estimate
// has end sooner. Measured, clusters and even (us): 32/32 heads of 64, trees of 5 rows: 1 behind 4,000 tokens 16 and 27, 4 behind 4,000 43 and 41, 16,000 152 and
// 100, 16 behind 250 16 and 18, 1,000 46 and 41, 64 behind 1,000 114 and 117; of 32 rows: 4 behind 1,000 21 and 31, 16,000 175 and 121. 32/8 heads of 128, trees of
// 1 row: 1 behind 16,000 53 and 43, 4 57 and 66, 16 200 and 185; of 8 rows: 1 61 and 71, 4 70 and 88, 16 242 and 230.
TreePlan tree_plan_mma(int num_seqs, int max_rows, int nh, int nkv, int hd, int max_context, int window, bool tc) {
    TreePlan p;
    const long long M = (long long)max_rows * (nh / nkv);
    if (tc && (hd == 64 || hd == 128) && window == 0 && tree_takes_tc(num_seqs, M, nkv, hd, max_context)) {
        p.tc = true;
        p.same = M <= TREE_TC_ROWS;
        p.blocks = 148;
        p.floats = ((long long)num_seqs * nkv * gb_ceil_div(M, p.same ? TREE_TC_ROWS : 2 * TREE_TC_ROWS) + p.blocks) * (p.same ? 1 : 2) * TREE_TC_ROWS * (hd + 2);
        return p;
    }
    p.rows = M <= 16 ? 16 : M <= 32 ? 32 : M <= 64 ? 64 : 128;
    const int room = 148 * (p.rows == 128 ? (hd > 64 ? 1 : 2) : hd > 64 ? 2 : hd == 64 ? 3 : 4);      // (as TmShape::BLOCKS)
    const long long items = (long long)num_seqs * nkv * gb_ceil_div(M, p.rows);
    const int reach = window > 0 && window + max_rows < max_context ? window + max_rows : max_context, tiles = gb_ceil_div(reach > 0 ? reach : 1, TM_KEYS);
    int c = TM_MAX_CLUSTER;
    while (c > 1 && (items * c > room || tiles < 2 * c)) c /= 2;
    const int even = hd == 64 && p.rows < 128 ? 148 * 4 : room;      // blocks of the even cut
    // microseconds of a tile in a block (what it waits for, or its share of a multiprocessor that moves 6.5 TB/s / 148 and multiplies 32 rows with 64 keys of 64
    // channels in 0.5), of a block's start, of the second launch, and of the pieces that it adds up
    auto tile_us = [&](long long blocks) {
        const double alone = 0.8 + hd / 160.0 + (p.rows > 16 ? 0.25 : 0.0), shared = hd / 64.0 * (p.rows > 16 ? p.rows / 64.0 : 0.37) * gb_ceil_div(blocks, 148);
        return alone > shared ? alone : shared;
    };
    const long long all = items * tiles, cut = gb_ceil_div(all, TREE_LEAST_SHARE) < even ? gb_ceil_div(all, TREE_LEAST_SHARE) : even;
    const double cluster_us = gb_ceil_div(items * c, room) * (gb_ceil_div(tiles, c) * tile_us(items * c < room ? items * c : room) + 6.0);
    const double even_us = gb_ceil_div(all, cut) * tile_us(cut) + 6.0 * items / cut + 20.0 + M / 4.0 + 0.3 * M / 16.0 * hd / 64.0 * cut / items;
    p.cluster = cluster_us <= even_us ? c : 0;
    p.blocks = p.cluster ? 0 : even;
    p.floats = p.cluster ? 0 : (items + even) * p.rows * (hd + 2);
    return p;
}
