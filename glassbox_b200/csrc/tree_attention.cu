// Attention of trees of drafted tokens over the paged cache, for every type, head size and page size: float32 arithmetic.
// (bfloat16 at the head sizes of tree_attention_mma.cu and tree_attention_tc.cu runs there.)
//
// A block takes 16 RT query rows of a request and key/value head over its share of the keys, 32 at a time from two buffers of shared memory, one of which is
// filled while the other is worked on. A thread forms the scores of RT rows and 4 keys, and the outputs of these rows at every eighth piece of four channels, so
// that a number from shared memory meets four others. Masks are looked at only in tiles that reach into the tree or out of a window; where one of these holds a
// value that is not a finite number, values go to the rows that see them one at a time, so that no weight of zero meets it. Shares of a request's keys that several
// blocks have go to the scratch as outputs, maximum and sum, and tree_merge_kernel adds them up.
//
// What bounds it: the multiply-adds, and the reads of shared memory that feed them (4 trees of 24 rows, 15/5 heads of 64, behind 1,500 tokens in float32: 57 us, 6
// TFLOP/s of multiply-adds); of few rows a block's chain.
#include "tree_attention.cuh"

constexpr int TA_THREADS = 128, TA_KEYS = 32, TA_MAX_HD = 256, TA_PP = TA_KEYS + 4;

template <typename T> __device__ __forceinline__ float4 ta_four(const T* p);
template <> __device__ __forceinline__ float4 ta_four<float>(const float* p) { return *reinterpret_cast<const float4*>(p); }
template <> __device__ __forceinline__ float4 ta_four<__nv_bfloat16>(const __nv_bfloat16* p) {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    return make_float4(__uint_as_float(v.x << 16), __uint_as_float(v.x & 0xffff0000u), __uint_as_float(v.y << 16), __uint_as_float(v.y & 0xffff0000u));
}
// Numbers of a row in shared memory: channels in fours (zeros behind the last), and 16 bytes so that eight rows' pieces lie in different banks.
template <typename T> static __host__ __device__ __forceinline__ int ta_pitch(int hd) { return (hd + 7) / 8 * 8 + 16 / (int)sizeof(T); }

template <typename T, int RT, int PIECES>      // rows of a thread; its pieces of four channels: hd <= 32 * PIECES
__global__ void __launch_bounds__(TA_THREADS) tree_attention_kernel(const TreeArgs a) {
    extern __shared__ __align__(16) unsigned char ta_smem[];
    constexpr int ROWS = 16 * RT;
    const int hd = a.hd, pitch = ta_pitch<T>(hd), qpitch = ta_pitch<float>(hd), fours = (hd + 3) / 4, tid = threadIdx.x, tx = tid & 7, ty = tid >> 3;
    float* Qs = reinterpret_cast<float*>(ta_smem);
    float* Ps = Qs + ROWS * qpitch;                   // [ROWS][TA_PP]
    T* KVs = reinterpret_cast<T*>(Ps + ROWS * TA_PP); // [2 buffers][keys, values][TA_KEYS][pitch]
    gb_pdl_launch_dependents();
    gb_pdl_wait();
    const TreeSeq s(a, blockIdx.z);
    const int G = a.nh / a.nkv, kvh = blockIdx.y % a.nkv, m0 = blockIdx.y / a.nkv * ROWS, M = s.rows * G, split = blockIdx.x;
    if (m0 >= M) return;
    T* out = (T*)a.out;
    if (s.start < 0) {                                // a padding request: zeros
        if (split == 0)
            for (int i = tid; i < min(ROWS, M - m0) * hd; i += TA_THREADS) {
                const int m = m0 + i / hd;
                out[(size_t)(s.row0 + m / G) * a.out_stride + (kvh * G + m % G) * hd + i % hd] = gb_from_float<T>(0.f);
            }
        return;
    }
    const int keys = s.length - s.key_lo, share = (keys + a.splits - 1) / a.splits, k_begin = s.key_lo + split * share, k_end = min(s.length, k_begin + share);
    const bool vec = hd * sizeof(T) % 16 == 0 && ((uintptr_t)a.kcache | (uintptr_t)a.vcache) % 16 == 0;
    bool bad = false;
    auto load = [&](int k0, int buffer) {             // 32 keys and values; zeros behind the share's last key
        T* to = KVs + buffer * 2 * TA_KEYS * pitch;
        if (vec) {
            const int pieces = hd * (int)sizeof(T) / 16;
            for (int i = tid; i < TA_KEYS * pieces; i += TA_THREADS) {
                const int r = i / pieces, c = i % pieces, key = k0 + r, page = key < k_end ? s.page(a, key / a.page_size) : -1;
                if (key < k_end && page < 0) bad = true;
                const size_t at = page < 0 ? 0 : (((size_t)page * a.nkv + kvh) * a.page_size + key % a.page_size) * hd * sizeof(T) + c * 16;
                const int bytes = page < 0 ? 0 : 16;
                const unsigned dst = (unsigned)__cvta_generic_to_shared(to + r * pitch) + c * 16;
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"((const char*)a.kcache + at), "r"(bytes) : "memory");
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst + TA_KEYS * pitch * (int)sizeof(T)), "l"((const char*)a.vcache + at), "r"(bytes) : "memory");
            }
        } else {
            for (int i = tid; i < TA_KEYS * 4 * fours; i += TA_THREADS) {
                const int r = i / (4 * fours), c = i % (4 * fours), key = k0 + r, page = key < k_end ? s.page(a, key / a.page_size) : -1;
                if (key < k_end && page < 0) bad = true;
                const size_t at = page < 0 ? 0 : (((size_t)page * a.nkv + kvh) * a.page_size + key % a.page_size) * hd + c;
                to[r * pitch + c] = page >= 0 && c < hd ? ((const T*)a.kcache)[at] : gb_from_float<T>(0.f);
                to[(TA_KEYS + r) * pitch + c] = page >= 0 && c < hd ? ((const T*)a.vcache)[at] : gb_from_float<T>(0.f);
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    if (k_begin < k_end) load(k_begin, 0);
    for (int i = tid; i < ROWS * 4 * fours; i += TA_THREADS) {
        const int r = i / (4 * fours), c = i % (4 * fours), m = m0 + r;
        Qs[r * qpitch + c] = m < M && c < hd ? gb_to_float(((const T*)a.q)[(size_t)(s.row0 + m / G) * a.q_stride + (kvh * G + m % G) * hd + c]) : 0.f;
    }
    // the thread's rows: RT ty ... of the tile
    int row[RT], pos[RT];
#pragma unroll
    for (int h = 0; h < RT; ++h) {
        const int m = m0 + RT * ty + h;
        row[h] = m < M ? s.row0 + m / G : -1;
        pos[h] = row[h] >= 0 ? a.positions[row[h]] : -1;
    }
    const float sl2 = a.scale * 1.4426950408889634f;
    float m_run[RT], l_run[RT], acc[RT][PIECES][4];
#pragma unroll
    for (int h = 0; h < RT; ++h) {
        m_run[h] = -INFINITY;
        l_run[h] = 0.f;
#pragma unroll
        for (int p = 0; p < PIECES; ++p)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[h][p][e] = 0.f;
    }
    for (int k0 = k_begin, buffer = 0; k0 < k_end; k0 += TA_KEYS, buffer ^= 1) {
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        __syncthreads();                              // the tile is there, the one before has been read
        if (k0 + TA_KEYS < k_end) load(k0 + TA_KEYS, buffer ^ 1);
        const T* Ks = KVs + buffer * 2 * TA_KEYS * pitch;
        const T* Vs = Ks + TA_KEYS * pitch;
        float sc[RT][4] = {};
        for (int c = 0; c < 4 * fours; c += 4) {
            float4 qv[RT], kv[4];
#pragma unroll
            for (int h = 0; h < RT; ++h) qv[h] = *reinterpret_cast<const float4*>(Qs + (RT * ty + h) * qpitch + c);
#pragma unroll
            for (int i = 0; i < 4; ++i) kv[i] = ta_four(Ks + (tx + 8 * i) * pitch + c);
#pragma unroll
            for (int h = 0; h < RT; ++h)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    sc[h][i] = fmaf(qv[h].x, kv[i].x, fmaf(qv[h].y, kv[i].y, fmaf(qv[h].z, kv[i].z, fmaf(qv[h].w, kv[i].w, sc[h][i]))));
        }
        const bool masked = k0 + TA_KEYS > min(s.start, k_end) || a.window > 0;      // (the same for the block)
        unsigned seen[RT];                            // of the tile's keys, by each of the rows
#pragma unroll
        for (int h = 0; h < RT; ++h) {
            float mx = -INFINITY;
            unsigned mine = 0xffffffffu;
            if (masked) {
                mine = row[h] < 0 ? 0u : tree_bits(a, s.rows, row[h], k0 - s.start);
                if (k_end - k0 < TA_KEYS) mine &= (1u << (k_end - k0)) - 1u;
                if (a.window > 0) {
                    unsigned near = 0u;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int key = k0 + tx + 8 * i;
                        if (mine >> (tx + 8 * i) & 1u)
                            near |= (unsigned)(pos[h] - (key < s.start ? key : a.positions[s.row0 + key - s.start]) < a.window) << (tx + 8 * i);
                    }
#pragma unroll
                    for (int o = 1; o < 8; o <<= 1) near |= __shfl_xor_sync(0xffffffffu, near, o);
                    mine = near;
                }
            }
            seen[h] = mine;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                sc[h][i] = mine >> (tx + 8 * i) & 1u ? sc[h][i] * sl2 : -INFINITY;
                mx = fmaxf(mx, sc[h][i]);
            }
#pragma unroll
            for (int o = 1; o < 8; o <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
            const float m_new = fmaxf(m_run[h], mx), off = m_new == -INFINITY ? 0.f : m_new, corr = exp2f(m_run[h] - off);
            m_run[h] = m_new;
            l_run[h] *= corr;
#pragma unroll
            for (int p = 0; p < PIECES; ++p)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[h][p][e] *= corr;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float p = exp2f(sc[h][i] - off);
                l_run[h] += p;
                Ps[(RT * ty + h) * TA_PP + tx + 8 * i] = p;
            }
        }
        // (a row's eight threads are neighbours; a value that is no finite number must not meet a weight of zero)
        bool odd = false;
        if (masked) {
            for (int i = tid; i < TA_KEYS * fours; i += TA_THREADS) {
                const float4 v = ta_four(Vs + i / fours * pitch + i % fours * 4);
                odd = odd || !isfinite(v.x) || !isfinite(v.y) || !isfinite(v.z) || !isfinite(v.w);
            }
            odd = __syncthreads_or(odd);
        } else {
            __syncwarp();
        }
        if (!odd) {
            for (int k = 0; k < TA_KEYS; k += 4) {
                float4 p4[RT];
#pragma unroll
                for (int h = 0; h < RT; ++h) p4[h] = *reinterpret_cast<const float4*>(Ps + (RT * ty + h) * TA_PP + k);
#pragma unroll
                for (int u = 0; u < 4; ++u)
#pragma unroll
                    for (int p = 0; p < PIECES; ++p) {
                        const int c = 4 * tx + 32 * p;
                        if (c >= hd) continue;
                        const float4 v = ta_four(Vs + (k + u) * pitch + c);
#pragma unroll
                        for (int h = 0; h < RT; ++h) {
                            const float w = u == 0 ? p4[h].x : u == 1 ? p4[h].y : u == 2 ? p4[h].z : p4[h].w;
                            acc[h][p][0] = fmaf(w, v.x, acc[h][p][0]);
                            acc[h][p][1] = fmaf(w, v.y, acc[h][p][1]);
                            acc[h][p][2] = fmaf(w, v.z, acc[h][p][2]);
                            acc[h][p][3] = fmaf(w, v.w, acc[h][p][3]);
                        }
                    }
            }
        } else {
            for (int k = 0; k < TA_KEYS; ++k)
#pragma unroll
                for (int h = 0; h < RT; ++h) {
                    if (!(seen[h] >> k & 1u)) continue;
                    const float w = Ps[(RT * ty + h) * TA_PP + k];
#pragma unroll
                    for (int p = 0; p < PIECES; ++p) {
                        const int c = 4 * tx + 32 * p;
                        if (c >= hd) continue;
                        const float4 v = ta_four(Vs + k * pitch + c);
                        acc[h][p][0] = fmaf(w, v.x, acc[h][p][0]);
                        acc[h][p][1] = fmaf(w, v.y, acc[h][p][1]);
                        acc[h][p][2] = fmaf(w, v.z, acc[h][p][2]);
                        acc[h][p][3] = fmaf(w, v.w, acc[h][p][3]);
                    }
                }
        }
    }
    if (bad) atomicOr(a.status, GB_STATUS_BAD_SLOT);
#pragma unroll
    for (int h = 0; h < RT; ++h) {
#pragma unroll
        for (int o = 1; o < 8; o <<= 1) l_run[h] += __shfl_xor_sync(0xffffffffu, l_run[h], o);
        if (row[h] < 0) continue;
        const int head = kvh * G + (m0 + RT * ty + h) % G;
        const size_t cell = (size_t)row[h] * a.nh + head, cells = (size_t)a.n * a.nh;
        float* part = a.parts + ((size_t)split * cells + cell) * hd;
        const float inv = l_run[h] != 0.f ? 1.0f / l_run[h] : 0.f;
#pragma unroll
        for (int p = 0; p < PIECES; ++p)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int c = 4 * tx + 32 * p + e;
                if (c >= hd) continue;
                if (a.splits == 1) out[(size_t)row[h] * a.out_stride + head * hd + c] = gb_from_float<T>(acc[h][p][e] * inv);
                else part[c] = acc[h][p][e];
            }
        if (a.splits > 1 && tx == 0)
            *reinterpret_cast<float2*>(a.parts + a.splits * cells * hd + ((size_t)split * cells + cell) * 2) = make_float2(m_run[h], l_run[h]);
    }
}

// Adds up the shares of a row and head: a warp each, a lane a share's weight.
template <typename T>
__global__ void __launch_bounds__(128) tree_merge_kernel(const TreeArgs a, int num_seqs) {
    gb_pdl_launch_dependents();
    gb_pdl_wait();
    const int lane = threadIdx.x & 31;
    const size_t cells = (size_t)a.n * a.nh, cell = (size_t)blockIdx.x * 4 + (threadIdx.x >> 5);
    if (cell >= cells) return;
    const int row = (int)(cell / a.nh);
    bool live = false;                                // the row belongs to a request that the shares are of (a padding request's rows have been written)
    for (int s0 = 0; s0 < num_seqs && !live; s0 += 32) {
        const int s = s0 + lane;
        live = __any_sync(0xffffffffu, s < num_seqs && a.start_pos[s] >= 0 && a.start_pos[s] <= a.places - tree_rows(a, s) && a.first_row[s] <= row &&
                                             row < a.first_row[s] + tree_rows(a, s));
    }
    if (!live) return;
    const float2* ml = reinterpret_cast<const float2*>(a.parts + a.splits * cells * a.hd) + cell;
    float top = -INFINITY;
    for (int i = lane; i < a.splits; i += 32) top = fmaxf(top, ml[i * cells].x);
    top = gb_warp_max(top);
    const float off = top == -INFINITY ? 0.f : top;
    float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}, l = 0.f;
    for (int i0 = 0; i0 < a.splits; i0 += 32) {
        const float2 own = i0 + lane < a.splits ? ml[(i0 + lane) * cells] : make_float2(-INFINITY, 0.f);
        const float f = exp2f(own.x - off);
        l = fmaf(own.y, f, l);
        const int count = min(32, a.splits - i0);
#pragma unroll 8
        for (int i = 0; i < count; ++i) {
            const float w = __shfl_sync(0xffffffffu, f, i);
            const float* part = a.parts + ((size_t)(i0 + i) * cells + cell) * a.hd;
#pragma unroll
            for (int c = 0; c < 8; ++c)
                if (lane + 32 * c < a.hd) v[c] = fmaf(part[lane + 32 * c], w, v[c]);
        }
    }
    l = gb_warp_sum(l);
    const float inv = l != 0.f ? 1.0f / l : 0.f;
#pragma unroll
    for (int c = 0; c < 8; ++c)
        if (lane + 32 * c < a.hd) ((T*)a.out)[(size_t)row * a.out_stride + (cell % a.nh) * a.hd + lane + 32 * c] = gb_from_float<T>(v[c] * inv);
}

// Query rows of a block, up to 48 (32 of heads above 128 channels, whose outputs fill the registers): those that leave few of them empty, and rather more, since
// the keys that a thread reads meet all of its rows. Measured in float32, blocks of 16 / 32 / 48 / 64 rows (us): 72 rows a request and key/value head, 4 requests
// of 15/5 heads of 64 behind 1,500 keys 75 / 68 / 67 / 103; 18 rows 43 / 39 / 43 / 66; 33 rows 53 / 54 / 46 / 70; 4 of 80 rows, 32/8 heads of 128, 200 / 174 / 157 / 178.
static int ta_rows(long long m, int hd) {
    int best = 16;
    double least = 0.0;
    for (int rows = 16; rows <= (hd > 128 ? 32 : 48); rows += 16) {
        const double cost = (double)gb_ceil_div(m, rows) * rows * (1.0 + 10.0 / rows);
        if (rows == 16 || cost < least) { best = rows; least = cost; }
    }
    return best;
}

template <typename T, int RT, int PIECES>
static int ta_launch(const TreeArgs& a, int num_seqs, int max_rows, cudaStream_t stream) {
    const int tiles = gb_ceil_div((long long)max_rows * (a.nh / a.nkv), 16 * RT);
    GB_REQUIRE((long long)tiles * a.nkv <= 65535, "gb_tree_attention: %d rows a request are too many for one launch", max_rows);
    const int smem = 16 * RT * (ta_pitch<float>(a.hd) + TA_PP) * 4 + 4 * TA_KEYS * ta_pitch<T>(a.hd) * (int)sizeof(T);
    cudaError_t e = cudaFuncSetAttribute(tree_attention_kernel<T, RT, PIECES>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    GB_REQUIRE(e == cudaSuccess, "gb_tree_attention: %d bytes of shared memory refused: %s", smem, cudaGetErrorString(e));
    e = gb_launch(GB_PDL_ATTENTION, tree_attention_kernel<T, RT, PIECES>, dim3(a.splits, tiles * a.nkv, num_seqs), dim3(TA_THREADS), smem, stream, a);
    GB_REQUIRE(e == cudaSuccess, "gb_tree_attention: launch failed: %s", cudaGetErrorString(e));
    return gb_check_launch("gb_tree_attention");
}

template <typename T, int PIECES>
static int ta_sized(const TreeArgs& a, int num_seqs, int max_rows, cudaStream_t stream) {
    const int rows = ta_rows((long long)max_rows * (a.nh / a.nkv), a.hd);
    if (rows == 16) return ta_launch<T, 1, PIECES>(a, num_seqs, max_rows, stream);
    if (rows == 32) return ta_launch<T, 2, PIECES>(a, num_seqs, max_rows, stream);
    if constexpr (PIECES <= 4) return ta_launch<T, 3, PIECES>(a, num_seqs, max_rows, stream);
    return 1;
}

template <typename T>
static int ta_dispatch(const TreeArgs& a, int num_seqs, int max_rows, cudaStream_t stream) {
    if (a.hd <= 64) return ta_sized<T, 2>(a, num_seqs, max_rows, stream);
    if (a.hd <= 128) return ta_sized<T, 4>(a, num_seqs, max_rows, stream);
    return ta_sized<T, 8>(a, num_seqs, max_rows, stream);
}

// tree_attention_mma.cu, tree_attention_tc.cu
int gb_tree_attention_tc(const TreeArgs& a, const TreePlan& plan, int num_seqs, int max_rows, cudaStream_t stream);
int gb_tree_attention_mma(const TreeArgs& a, const TreePlan& plan, int num_seqs, int max_rows, cudaStream_t stream);
TreePlan tree_plan_mma(int num_seqs, int max_rows, int nh, int nkv, int hd, int max_context, int window, bool tc);

// Shares of a request's keys in this file's kernel, so that blocks fill the GPU, of 64 keys at least.
static int ta_splits(int num_seqs, int max_rows, int nh, int nkv, int hd, int max_context, int window) {
    const long long m = (long long)max_rows * (nh / nkv), blocks = (long long)num_seqs * nkv * gb_ceil_div(m, ta_rows(m, hd));
    const int reach = window > 0 && window + max_rows < max_context ? window + max_rows : max_context, most = reach <= 64 ? 1 : gb_ceil_div(reach, 64);
    const long long splits = 148ll * 4 / blocks;
    return splits > most ? most : splits < 1 ? 1 : (int)splits;
}

// Numbers (float32) of the scratch that a call needs; -1: more than there can be. kind as below.
GB_EXPORT int gb_tree_attention_floats(int kind, int n, int num_seqs, int max_rows, int nh, int nkv, int hd, int max_context, int window) {
    if (n <= 0 || num_seqs <= 0 || max_rows <= 0 || nkv <= 0 || nh % nkv) return 0;
    long long floats;
    if (kind >= 1) {
        floats = tree_plan_mma(num_seqs, max_rows, nh, nkv, hd, max_context, window, kind == 2).floats;
    } else {
        const int splits = ta_splits(num_seqs, max_rows, nh, nkv, hd, max_context, window);
        floats = splits > 1 ? (long long)splits * n * nh * (hd + 2) : 0;
    }
    return floats < (1ll << 31) ? (int)floats : -1;
}

// kind 0: this file's kernel; 1: the tensor cores (bfloat16); 2: tcgen05 where there is enough for it (scale above 0, pages of 8 to 128, rows of q and out at 16 bytes). q, out: [n, nh * hd], rows `stride` numbers apart; kcache, vcache: [num_pages, nkv, page_size, hd];
// parts: gb_tree_attention_floats of the same sizes.
GB_EXPORT int gb_tree_attention(int kind, const void* q, long long q_stride, void* out, long long out_stride, int dtype, const void* kcache, const void* vcache,
                                const int* block_tables, int max_pages, const int* first_row, const int* start_pos, const int* positions, const int* visible,
                                int words, int n, int num_seqs, int max_rows, int nh, int nkv, int hd, int page_size, long long num_pages, float scale,
                                int window, int max_context, float* parts, int* status, cudaStream_t stream) {
    GB_REQUIRE(nkv > 0 && nh > 0 && nh % nkv == 0 && hd > 0 && hd <= TA_MAX_HD, "gb_tree_attention: %d/%d heads of %d are not built", nh, nkv, hd);
    GB_REQUIRE(n >= 0 && num_seqs >= 0 && num_seqs <= 65535 && max_rows >= 0 && max_pages > 0 && page_size > 0 && num_pages > 0 && words > 0 && window >= 0,
               "gb_tree_attention: bad batch shape");
    GB_REQUIRE(dtype == GB_F32 || dtype == GB_BF16, "gb_tree_attention: unsupported dtype %d", dtype);
    GB_REQUIRE((long long)max_pages * page_size < (1ll << 31) - 4096, "gb_tree_attention: the block tables reach too far");
    if (n == 0 || num_seqs == 0 || max_rows == 0) return 0;
    GB_REQUIRE(q && out && kcache && vcache && block_tables && first_row && start_pos && positions && visible && status, "gb_tree_attention: a tensor is missing");
    TreeArgs a = {q, q_stride, out, out_stride, kcache, vcache, block_tables, max_pages, max_pages * page_size, first_row, start_pos, positions, visible, words, n, max_rows, nh, nkv, hd, page_size,
                  num_pages, scale, window, 1, parts, status};
    if (kind >= 1) {
        GB_REQUIRE(kind == 1 || (scale > 0.f && page_size >= 8 && page_size <= TREE_TC_KEYS && (uintptr_t)q % 16 == 0 && q_stride % 8 == 0 && (uintptr_t)out % 16 == 0 && out_stride % 8 == 0),
                   "gb_tree_attention: this scale, page size or alignment is not built for tcgen05");
        GB_REQUIRE(dtype == GB_BF16, "gb_tree_attention: the tensor cores' kernel takes bfloat16");
        const TreePlan plan = tree_plan_mma(num_seqs, max_rows, nh, nkv, hd, max_context, window, kind == 2);
        GB_REQUIRE(plan.floats == 0 || (parts != nullptr && (uintptr_t)parts % 16 == 0), "gb_tree_attention: the scratch is missing or not 16-byte aligned");
        return plan.tc ? gb_tree_attention_tc(a, plan, num_seqs, max_rows, stream) : gb_tree_attention_mma(a, plan, num_seqs, max_rows, stream);
    }
    a.splits = ta_splits(num_seqs, max_rows, nh, nkv, hd, max_context, window);
    GB_REQUIRE(a.splits == 1 || parts != nullptr, "gb_tree_attention: the scratch is missing");
    const int rc = dtype == GB_F32 ? ta_dispatch<float>(a, num_seqs, max_rows, stream) : ta_dispatch<__nv_bfloat16>(a, num_seqs, max_rows, stream);
    if (rc || a.splits == 1) return rc;
    const unsigned blocks = (unsigned)(((size_t)n * nh + 3) / 4);
    const cudaError_t e = dtype == GB_F32 ? gb_launch(GB_PDL_ATTENTION, tree_merge_kernel<float>, dim3(blocks), dim3(128), 0, stream, a, num_seqs)
                                          : gb_launch(GB_PDL_ATTENTION, tree_merge_kernel<__nv_bfloat16>, dim3(blocks), dim3(128), 0, stream, a, num_seqs);
    GB_REQUIRE(e == cudaSuccess, "gb_tree_attention: launch failed: %s", cudaGetErrorString(e));
    return gb_check_launch("gb_tree_attention");
}
