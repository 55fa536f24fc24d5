// Attention of trees of drafted tokens over the paged cache in bfloat16 on the tensor cores (mma.sync m16n8k16), head sizes 32, 64, 96 and 128.
//
// A block takes 16 WM query rows (rows of the tree x query heads that share the key/value head) of a request over its share of the keys, 64 at a time
// through a ring of three stages that asynchronous copies fill; WM x WK warps, each with 16 of the rows and 64 / WK of a stage's keys, so that small trees
// keep four warps at work. Rows of shared memory are padded by 16 bytes: eight rows' pieces lie in different banks. Softmax statistics and outputs are
// float32 (a maximum and a sum per row and warp, added up at the end); weights are rounded to bfloat16 on their way into the second product, 2^-9 of each.
//
// Masks are looked at only where a warp's keys hold some that a row may not see: bits of the tree come as 32 at a time. There a value that is not a finite
// number must not meet a weight of zero, so such keys go one by one.
#include "tree_attention.cuh"

constexpr int TM_KEYS = 64, TM_STAGES = 3, TM_MAX_PAGES = 1024;

__device__ __forceinline__ uint32_t tm_smem(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
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

// Of the 32 rows of the tree from d0 on (negative: keys before the tree, all seen), those that a row of the batch sees.
__device__ __forceinline__ unsigned tm_bits(const TreeArgs& a, int rows, int row, int d0) {
    if (d0 <= -32) return 0xffffffffu;
    if (row < 0) return 0u;
    const unsigned* bits = reinterpret_cast<const unsigned*>(a.visible) + (size_t)row * a.words;
    unsigned v;
    if (d0 < 0) {
        v = ((1u << -d0) - 1u) | (bits[0] << -d0);
    } else {
        const int w = d0 >> 5, sh = d0 & 31;
        v = w < a.words ? bits[w] >> sh : 0u;
        if (sh && w + 1 < a.words) v |= bits[w + 1] << (32 - sh);
    }
    const int left = rows - d0;
    return left >= 32 ? v : left <= 0 ? 0u : v & ((1u << left) - 1u);
}

template <int HD, int WM, int WK>
struct TmShape {
    static constexpr int PITCH = HD * 2 + 16, TILE = TM_KEYS * PITCH, THREADS = WM * WK * 32, ROWS = WM * 16, KW = TM_KEYS / WK;
    static constexpr int SMEM = 2 * TM_STAGES * TILE + TM_MAX_PAGES * 4;
    static_assert(WK == 1 || WM * WK * 16 * (HD + 2) * 4 <= 2 * TM_STAGES * TILE, "the warps' results lie over the stages");
};

template <int HD, int WM, int WK>
__global__ void __launch_bounds__(WM* WK * 32) tree_attention_mma_kernel(const TreeArgs a) {
    using Sh = TmShape<HD, WM, WK>;
    constexpr int CH = HD / 8, KS = HD / 16, NT = HD / 8, KW = Sh::KW, KT = KW / 8;
    extern __shared__ __align__(16) unsigned char tm_mem[];
    unsigned char* Ks = tm_mem;
    unsigned char* Vs = tm_mem + TM_STAGES * Sh::TILE;
    int* pages = reinterpret_cast<int*>(tm_mem + 2 * TM_STAGES * Sh::TILE);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, wm = warp % WM, wk = warp / WM, g = lane >> 2, t = lane & 3;
    const int G = a.nh / a.nkv, kvh = blockIdx.y % a.nkv, m0 = blockIdx.y / a.nkv * Sh::ROWS, split = blockIdx.x;
    gb_pdl_launch_dependents();
    gb_pdl_wait();
    const TreeSeq s(a, blockIdx.z);
    const int M = s.rows * G;
    if (m0 >= M) return;
    __nv_bfloat16* out = (__nv_bfloat16*)a.out;
    // the thread's two rows: g and g + 8 of the warp's
    int row[2], head[2], pos[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int m = m0 + wm * 16 + g + 8 * h;
        row[h] = m < M ? s.row0 + m / G : -1;
        head[h] = kvh * G + m % G;
        pos[h] = row[h] >= 0 ? a.positions[row[h]] : -1;
    }
    if (s.start < 0) {                                // a padding request: zeros
        if (split == 0 && wk == 0)
            for (int h = 0; h < 2; ++h)
                for (int c = 2 * t; row[h] >= 0 && c < HD; c += 8) *reinterpret_cast<uint32_t*>(out + (size_t)row[h] * a.out_stride + head[h] * HD + c) = 0u;
        return;
    }
    const int base = s.key_lo / TM_KEYS * TM_KEYS, share = ((s.length - base + a.splits - 1) / a.splits + TM_KEYS - 1) / TM_KEYS * TM_KEYS;
    const int k_begin = min(s.length, base + split * share), k_end = min(s.length, k_begin + share);
    const int tiles = (k_end - k_begin + TM_KEYS - 1) / TM_KEYS;
    int shift = 0;
    while ((1 << shift) < a.page_size) ++shift;
    const int page_lo = k_begin >> shift, n_pages = tiles ? ((k_end - 1) >> shift) - page_lo + 1 : 0;
    const bool staged = n_pages <= TM_MAX_PAGES;
    bool bad = false;
    if (staged)
        for (int i = tid; i < n_pages; i += Sh::THREADS) pages[i] = s.page(a, page_lo + i);
    uint32_t qf[KS][4];
#pragma unroll
    for (int k = 0; k < KS; ++k)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int h = i & 1;
            qf[k][i] = row[h] >= 0 ? *reinterpret_cast<const uint32_t*>((const __nv_bfloat16*)a.q + (size_t)row[h] * a.q_stride + head[h] * HD + 16 * k + 8 * (i >> 1) + 2 * t) : 0u;
        }
    __syncthreads();

    const __nv_bfloat16* kc = (const __nv_bfloat16*)a.kcache;
    const __nv_bfloat16* vc = (const __nv_bfloat16*)a.vcache;
    auto load = [&](int tile) {
        const int k0 = k_begin + tile * TM_KEYS, stage = tile % TM_STAGES;
        const uint32_t kb = tm_smem(Ks + stage * Sh::TILE), vb = tm_smem(Vs + stage * Sh::TILE);
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
#pragma unroll
    for (int i = 0; i < TM_STAGES - 1; ++i) {
        if (i < tiles) load(i);
        asm volatile("cp.async.commit_group;" ::: "memory");
    }
    const float sl2 = a.scale * 1.4426950408889634f;
    float m_run[2] = {-INFINITY, -INFINITY}, l_run[2] = {0.f, 0.f}, acc[NT][4];
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[j][e] = 0.f;
    for (int tile = 0; tile < tiles; ++tile) {
        asm volatile("cp.async.wait_group %0;" ::"n"(TM_STAGES - 2) : "memory");
        __syncthreads();                              // the tile is there, and the one before has been read
        if (tile + TM_STAGES - 1 < tiles) load(tile + TM_STAGES - 1);
        asm volatile("cp.async.commit_group;" ::: "memory");
        const int k0 = k_begin + tile * TM_KEYS + wk * KW;      // of the warp's keys
        const unsigned char* vs = Vs + (tile % TM_STAGES) * Sh::TILE + wk * KW * Sh::PITCH;
        const uint32_t kb = tm_smem(Ks + (tile % TM_STAGES) * Sh::TILE) + (wk * KW + (lane >> 4) * 8 + (lane & 7)) * Sh::PITCH + ((lane >> 3) & 1) * 16;
        const uint32_t vb = tm_smem(vs) + (((lane >> 3) & 1) * 8 + (lane & 7)) * Sh::PITCH + (lane >> 4) * 16;
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
                tm_ldmatrix(b, kb + j * 8 * Sh::PITCH + k * 32);
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
                for (int w = 0; w < (KW + 31) / 32; ++w) see[h][w] = tm_bits(a, s.rows, row[h], k0 + 32 * w - s.start);
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
                const uint4 v = *reinterpret_cast<const uint4*>(vs + i / CH * Sh::PITCH + i % CH * 16);
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
        if (!odd) {
#pragma unroll
            for (int b = 0; b < KW / 16; ++b) {
                const uint32_t p[4] = {tm_pack(sc[2 * b][0], sc[2 * b][1]), tm_pack(sc[2 * b][2], sc[2 * b][3]), tm_pack(sc[2 * b + 1][0], sc[2 * b + 1][1]),
                                       tm_pack(sc[2 * b + 1][2], sc[2 * b + 1][3])};
#pragma unroll
                for (int j = 0; j < NT; j += 2) {
                    uint32_t v[4];
                    tm_ldmatrix_t(v, vb + b * 16 * Sh::PITCH + j * 16);
                    tm_mma(acc[j], p, v[0], v[1]);
                    tm_mma(acc[j + 1], p, v[2], v[3]);
                }
            }
        } else {
#pragma unroll
            for (int j = 0; j < KT; ++j)
#pragma unroll
                for (int e = 0; e < 2; ++e)
                    for (int tt = 0; tt < 4; ++tt) {
                        const float p0 = __shfl_sync(0xffffffffu, sc[j][e], (lane & ~3) | tt), p1 = __shfl_sync(0xffffffffu, sc[j][2 + e], (lane & ~3) | tt);
                        const unsigned char* v = vs + (8 * j + 2 * tt + e) * Sh::PITCH + 4 * t;
#pragma unroll
                        for (int c = 0; c < NT; ++c) {
                            const uint32_t two = *reinterpret_cast<const uint32_t*>(v + 16 * c);
                            const float lo = __uint_as_float(two << 16), hi = __uint_as_float(two & 0xffff0000u);
                            if (p0 != 0.f) { acc[c][0] = fmaf(p0, lo, acc[c][0]); acc[c][1] = fmaf(p0, hi, acc[c][1]); }
                            if (p1 != 0.f) { acc[c][2] = fmaf(p1, lo, acc[c][2]); acc[c][3] = fmaf(p1, hi, acc[c][3]); }
                        }
                    }
        }
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    if (bad) atomicOr(a.status, GB_STATUS_BAD_SLOT);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        l_run[h] += __shfl_xor_sync(0xffffffffu, l_run[h], 1);
        l_run[h] += __shfl_xor_sync(0xffffffffu, l_run[h], 2);
    }
    const size_t cells = (size_t)a.n * a.nh;
    float* stats = a.parts + a.splits * cells * HD;
    if constexpr (WK == 1) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            if (row[h] < 0) continue;
            const size_t cell = (size_t)row[h] * a.nh + head[h];
            if (a.splits == 1) {
                const float inv = l_run[h] != 0.f ? 1.0f / l_run[h] : 0.f;
#pragma unroll
                for (int j = 0; j < NT; ++j)
                    *reinterpret_cast<uint32_t*>(out + (size_t)row[h] * a.out_stride + head[h] * HD + 8 * j + 2 * t) = tm_pack(acc[j][2 * h] * inv, acc[j][2 * h + 1] * inv);
            } else {
                float* part = a.parts + ((size_t)split * cells + cell) * HD;
#pragma unroll
                for (int j = 0; j < NT; ++j) *reinterpret_cast<float2*>(part + 8 * j + 2 * t) = make_float2(acc[j][2 * h], acc[j][2 * h + 1]);
                if (t == 0) *reinterpret_cast<float2*>(stats + ((size_t)split * cells + cell) * 2) = make_float2(m_run[h], l_run[h]);
            }
        }
    } else {
        constexpr int P = HD + 2;                     // a warp's result of a row: channels, maximum, sum
        float* res = reinterpret_cast<float*>(tm_mem);
        __syncthreads();                              // (all stages have been read)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            float* to = res + ((size_t)(wk * WM + wm) * 16 + g + 8 * h) * P;
#pragma unroll
            for (int j = 0; j < NT; ++j) *reinterpret_cast<float2*>(to + 8 * j + 2 * t) = make_float2(acc[j][2 * h], acc[j][2 * h + 1]);
            if (t == 0) *reinterpret_cast<float2*>(to + HD) = make_float2(m_run[h], l_run[h]);
        }
        __syncthreads();
        for (int i = tid; i < Sh::ROWS * (HD / 2); i += Sh::THREADS) {
            const int r = i / (HD / 2), c = i % (HD / 2) * 2, m = m0 + r;
            if (m >= M) break;
            float top = -INFINITY, l = 0.f, x = 0.f, y = 0.f;
#pragma unroll
            for (int w = 0; w < WK; ++w) top = fmaxf(top, res[((size_t)w * Sh::ROWS + r) * P + HD]);
            const float o = top == -INFINITY ? 0.f : top;
#pragma unroll
            for (int w = 0; w < WK; ++w) {
                const float* from = res + ((size_t)w * Sh::ROWS + r) * P;
                const float f = tm_exp2(from[HD] - o);
                l = fmaf(from[HD + 1], f, l);
                x = fmaf(from[c], f, x);
                y = fmaf(from[c + 1], f, y);
            }
            const int to_row = s.row0 + m / G, to_head = kvh * G + m % G;
            const size_t cell = (size_t)to_row * a.nh + to_head;
            if (a.splits == 1) {
                const float inv = l != 0.f ? 1.0f / l : 0.f;
                *reinterpret_cast<uint32_t*>(out + (size_t)to_row * a.out_stride + to_head * HD + c) = tm_pack(x * inv, y * inv);
            } else {
                *reinterpret_cast<float2*>(a.parts + ((size_t)split * cells + cell) * HD + c) = make_float2(x, y);
                if (c == 0) *reinterpret_cast<float2*>(stats + ((size_t)split * cells + cell) * 2) = make_float2(top, l);
            }
        }
    }
}

template <int HD, int WM, int WK>
static int tm_launch(const TreeArgs& a, int num_seqs, int max_rows, cudaStream_t stream) {
    using Sh = TmShape<HD, WM, WK>;
    const int tiles = gb_ceil_div((long long)max_rows * (a.nh / a.nkv), Sh::ROWS);
    GB_REQUIRE((long long)tiles * a.nkv <= 65535, "gb_tree_attention: %d rows a request are too many for one launch", max_rows);
    cudaError_t e = cudaFuncSetAttribute(tree_attention_mma_kernel<HD, WM, WK>, cudaFuncAttributeMaxDynamicSharedMemorySize, Sh::SMEM);
    GB_REQUIRE(e == cudaSuccess, "gb_tree_attention: %d bytes of shared memory refused: %s", Sh::SMEM, cudaGetErrorString(e));
    e = gb_launch(GB_PDL_ATTENTION, tree_attention_mma_kernel<HD, WM, WK>, dim3(a.splits, tiles * a.nkv, num_seqs), dim3(Sh::THREADS), Sh::SMEM, stream, a);
    GB_REQUIRE(e == cudaSuccess, "gb_tree_attention: launch failed: %s", cudaGetErrorString(e));
    return gb_check_launch("gb_tree_attention");
}

template <int HD>
static int tm_dispatch(const TreeArgs& a, int num_seqs, int max_rows, cudaStream_t stream) {
    const long long M = (long long)max_rows * (a.nh / a.nkv);
    if (M <= 16) return tm_launch<HD, 1, 4>(a, num_seqs, max_rows, stream);
    if (M <= 32) return tm_launch<HD, 2, 2>(a, num_seqs, max_rows, stream);
    if (M <= 64) return tm_launch<HD, 4, 1>(a, num_seqs, max_rows, stream);
    return tm_launch<HD, 8, 1>(a, num_seqs, max_rows, stream);
}

int gb_tree_attention_mma(const TreeArgs& a, int num_seqs, int max_rows, cudaStream_t stream) {
    GB_REQUIRE(a.page_size > 0 && (a.page_size & (a.page_size - 1)) == 0, "gb_tree_attention: pages of %d tokens (a power of two) are not built here", a.page_size);
    GB_REQUIRE((uintptr_t)a.kcache % 16 == 0 && (uintptr_t)a.vcache % 16 == 0 && (uintptr_t)a.q % 4 == 0 && a.q_stride % 2 == 0 && (uintptr_t)a.out % 4 == 0 && a.out_stride % 2 == 0,
               "gb_tree_attention: rows must be 4-byte aligned, pages 16-byte aligned");
    if (a.hd == 32) return tm_dispatch<32>(a, num_seqs, max_rows, stream);
    if (a.hd == 64) return tm_dispatch<64>(a, num_seqs, max_rows, stream);
    if (a.hd == 96) return tm_dispatch<96>(a, num_seqs, max_rows, stream);
    GB_REQUIRE(a.hd == 128, "gb_tree_attention: heads of %d are not built here", a.hd);
    return tm_dispatch<128>(a, num_seqs, max_rows, stream);
}

// How many shares the keys of a request are cut into, for the kernels of gb_tree_attention (kind as there).
GB_EXPORT int gb_tree_attention_splits(int kind, int num_seqs, int max_rows, int nh, int nkv, int hd, int max_context, int window) {
    if (num_seqs <= 0 || max_rows <= 0 || nkv <= 0) return 1;
    const long long M = (long long)max_rows * (nh / nkv);
    const int rows = kind == 0 ? 32 : M <= 16 ? 16 : M <= 32 ? 32 : M <= 64 ? 64 : 128;
    const long long blocks = (long long)num_seqs * nkv * gb_ceil_div(M, rows);
    const int reach = window > 0 && window + max_rows < max_context ? window + max_rows : max_context;
    const int least = kind == 0 ? 128 : 256, most = reach <= least ? 1 : gb_ceil_div(reach, least);
    const long long room = 148ll * (hd > 96 ? 2 : 3);
    long long splits = room / blocks;
    if (splits > most) splits = most;
    return splits < 1 ? 1 : (int)splits;
}
