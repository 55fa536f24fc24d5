// Attention of trees of drafted tokens over the paged cache, for every type, head size and page size: float32 arithmetic.
// (bfloat16 at the head sizes of tree_attention_mma.cu runs there.)
//
// A block takes 32 query rows of a request and key/value head over its share of the keys, 32 at a time from shared memory; a thread forms the scores of
// 2 rows and 4 keys, and the outputs of the 2 rows at every eighth piece of four channels. What is masked never enters a sum: its weight is not formed.
#include "tree_attention.cuh"

constexpr int TA_THREADS = 128, TA_ROWS = 32, TA_KEYS = 32, TA_MAX_HD = 256;

static __host__ __device__ __forceinline__ int ta_pitch(int hd) { return (hd + 3) / 4 * 4 + 4; }      // floats of a row in shared memory

template <typename T, int PIECES>      // pieces of four channels of a thread: hd <= 32 * PIECES
__global__ void __launch_bounds__(TA_THREADS) tree_attention_kernel(const TreeArgs a) {
    extern __shared__ __align__(16) float ta_smem[];
    const int hd = a.hd, pitch = ta_pitch(hd), tid = threadIdx.x, tx = tid & 7, ty = tid >> 3;
    float* Qs = ta_smem;
    float* Ks = Qs + TA_ROWS * pitch;
    float* Vs = Ks + TA_KEYS * pitch;
    float* Ps = Vs + TA_KEYS * pitch;                 // [TA_ROWS][TA_KEYS + 1]
    gb_pdl_launch_dependents();
    gb_pdl_wait();
    const TreeSeq s(a, blockIdx.z);
    const int G = a.nh / a.nkv, kvh = blockIdx.y % a.nkv, m0 = blockIdx.y / a.nkv * TA_ROWS, M = s.rows * G, split = blockIdx.x;
    if (m0 >= M) return;
    T* out = (T*)a.out;
    // the thread's two rows: 2 ty and 2 ty + 1 of the tile
    int row[2], head[2], pos[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int m = m0 + 2 * ty + h;
        row[h] = m < M ? s.row0 + m / G : -1;
        head[h] = kvh * G + m % G;
        pos[h] = row[h] >= 0 ? a.positions[row[h]] : -1;
    }
    if (s.start < 0) {                                // a padding request: zeros
        if (split == 0)
            for (int h = 0; h < 2; ++h)
                for (int c = tx; row[h] >= 0 && c < hd; c += 8) out[(size_t)row[h] * a.out_stride + head[h] * hd + c] = gb_from_float<T>(0.f);
        return;
    }
    const int keys = s.length - s.key_lo, share = (keys + a.splits - 1) / a.splits, k_begin = s.key_lo + split * share, k_end = min(s.length, k_begin + share);
    for (int i = tid; i < TA_ROWS * pitch; i += TA_THREADS) {
        const int m = m0 + i / pitch, c = i % pitch;
        Qs[i] = m < M && c < hd ? gb_to_float(((const T*)a.q)[(size_t)(s.row0 + m / G) * a.q_stride + (kvh * G + m % G) * hd + c]) : 0.f;
    }
    const float sl2 = a.scale * 1.4426950408889634f;
    float m_run[2] = {-INFINITY, -INFINITY}, l_run[2] = {0.f, 0.f}, acc[2][PIECES][4];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int p = 0; p < PIECES; ++p)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[h][p][e] = 0.f;
    bool bad = false;
    for (int k0 = k_begin; k0 < k_end; k0 += TA_KEYS) {
        __syncthreads();                              // (the tile before has been read)
        for (int i = tid; i < TA_KEYS * pitch; i += TA_THREADS) {
            const int key = k0 + i / pitch, c = i % pitch;
            float kv = 0.f, vv = 0.f;
            if (key < k_end && c < hd) {
                const int page = s.page(a, key / a.page_size);
                if (page >= 0) {
                    const size_t at = (((size_t)page * a.nkv + kvh) * a.page_size + key % a.page_size) * hd + c;
                    kv = gb_to_float(((const T*)a.kcache)[at]);
                    vv = gb_to_float(((const T*)a.vcache)[at]);
                } else {
                    bad = true;
                }
            }
            Ks[i] = kv;
            Vs[i] = vv;
        }
        __syncthreads();
        float sc[2][4] = {};
        for (int c = 0; c < pitch - 4; c += 4) {
            float4 qv[2], kv[4];
#pragma unroll
            for (int h = 0; h < 2; ++h) qv[h] = *reinterpret_cast<const float4*>(Qs + (2 * ty + h) * pitch + c);
#pragma unroll
            for (int i = 0; i < 4; ++i) kv[i] = *reinterpret_cast<const float4*>(Ks + (tx + 8 * i) * pitch + c);
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    sc[h][i] = fmaf(qv[h].x, kv[i].x, fmaf(qv[h].y, kv[i].y, fmaf(qv[h].z, kv[i].z, fmaf(qv[h].w, kv[i].w, sc[h][i]))));
        }
        const bool masked = k0 + TA_KEYS > min(s.start, k_end) || a.window > 0;
        unsigned seen[2];                             // of the tile's keys, for each of the two rows
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            float mx = -INFINITY;
            unsigned mine = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int key = k0 + tx + 8 * i;
                const bool ok = row[h] >= 0 && (!masked || (key < k_end && s.sees(a, row[h], pos[h], key)));
                mine |= (unsigned)ok << (tx + 8 * i);
                sc[h][i] *= sl2;
                if (ok) mx = fmaxf(mx, sc[h][i]);
            }
#pragma unroll
            for (int o = 1; o < 8; o <<= 1) {
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
                mine |= __shfl_xor_sync(0xffffffffu, mine, o);
            }
            seen[h] = mine;
            const float m_new = fmaxf(m_run[h], mx), off = m_new == -INFINITY ? 0.f : m_new, corr = exp2f(m_run[h] - off);
            m_run[h] = m_new;
            l_run[h] *= corr;
#pragma unroll
            for (int p = 0; p < PIECES; ++p)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[h][p][e] *= corr;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float p = mine >> (tx + 8 * i) & 1u ? exp2f(sc[h][i] - off) : 0.f;
                l_run[h] += p;
                Ps[(2 * ty + h) * (TA_KEYS + 1) + tx + 8 * i] = p;
            }
        }
        __syncwarp();                                 // (a row's eight threads are neighbours)
        const unsigned either = seen[0] | seen[1];
        for (int k = 0; k < TA_KEYS; ++k) {
            if (!(either >> k & 1u)) continue;
            const float p0 = Ps[(2 * ty) * (TA_KEYS + 1) + k], p1 = Ps[(2 * ty + 1) * (TA_KEYS + 1) + k];
            const bool s0 = seen[0] >> k & 1u, s1 = seen[1] >> k & 1u;
#pragma unroll
            for (int p = 0; p < PIECES; ++p) {
                const int c = 4 * tx + 32 * p;
                if (c >= hd) continue;
                const float4 v = *reinterpret_cast<const float4*>(Vs + k * pitch + c);
                if (s0) { acc[0][p][0] = fmaf(p0, v.x, acc[0][p][0]); acc[0][p][1] = fmaf(p0, v.y, acc[0][p][1]); acc[0][p][2] = fmaf(p0, v.z, acc[0][p][2]); acc[0][p][3] = fmaf(p0, v.w, acc[0][p][3]); }
                if (s1) { acc[1][p][0] = fmaf(p1, v.x, acc[1][p][0]); acc[1][p][1] = fmaf(p1, v.y, acc[1][p][1]); acc[1][p][2] = fmaf(p1, v.z, acc[1][p][2]); acc[1][p][3] = fmaf(p1, v.w, acc[1][p][3]); }
            }
        }
    }
    if (bad) atomicOr(a.status, GB_STATUS_BAD_SLOT);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int o = 1; o < 8; o <<= 1) l_run[h] += __shfl_xor_sync(0xffffffffu, l_run[h], o);
        if (row[h] < 0) continue;
        const size_t cell = (size_t)row[h] * a.nh + head[h], cells = (size_t)a.n * a.nh;
        float* part = a.parts + ((size_t)split * cells + cell) * hd;
        const float inv = l_run[h] != 0.f ? 1.0f / l_run[h] : 0.f;
#pragma unroll
        for (int p = 0; p < PIECES; ++p)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int c = 4 * tx + 32 * p + e;
                if (c >= hd) continue;
                if (a.splits == 1) out[(size_t)row[h] * a.out_stride + head[h] * hd + c] = gb_from_float<T>(acc[h][p][e] * inv);
                else part[c] = acc[h][p][e];
            }
        if (a.splits > 1 && tx == 0)
            *reinterpret_cast<float2*>(a.parts + a.splits * cells * hd + ((size_t)split * cells + cell) * 2) = make_float2(m_run[h], l_run[h]);
    }
}

// Adds up the shares of a row and head: a warp each.
template <typename T>
__global__ void __launch_bounds__(128) tree_merge_kernel(const TreeArgs a, int num_seqs) {
    gb_pdl_launch_dependents();
    gb_pdl_wait();
    const int lane = threadIdx.x & 31;
    const size_t cells = (size_t)a.n * a.nh, cell = (size_t)blockIdx.x * 4 + (threadIdx.x >> 5);
    const int row = (int)(cell / a.nh);
    if (cell >= cells || row < a.first_row[0] || row >= a.first_row[num_seqs]) return;
    int lo = 0, hi = num_seqs;                        // the row's request: a padding one has been written
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (a.first_row[mid] <= row) lo = mid; else hi = mid;
    }
    if (a.start_pos[lo] < 0) return;
    const float2* ml = reinterpret_cast<const float2*>(a.parts + a.splits * cells * a.hd) + cell;
    float m = -INFINITY, l = 0.f;
    for (int i = 0; i < a.splits; ++i) m = fmaxf(m, ml[i * cells].x);
    const float off = m == -INFINITY ? 0.f : m;
    for (int i = 0; i < a.splits; ++i) l = fmaf(ml[i * cells].y, exp2f(ml[i * cells].x - off), l);
    const float inv = l != 0.f ? 1.0f / l : 0.f;
    for (int c = lane; c < a.hd; c += 32) {
        float v = 0.f;
#pragma unroll 4
        for (int i = 0; i < a.splits; ++i) v = fmaf(a.parts[(i * cells + cell) * a.hd + c], exp2f(ml[i * cells].x - off), v);
        ((T*)a.out)[(size_t)row * a.out_stride + (cell % a.nh) * a.hd + c] = gb_from_float<T>(v * inv);
    }
}

template <typename T, int PIECES>
static int ta_launch(const TreeArgs& a, int num_seqs, int tiles, cudaStream_t stream) {
    const int smem = ((TA_ROWS + 2 * TA_KEYS) * ta_pitch(a.hd) + TA_ROWS * (TA_KEYS + 1)) * (int)sizeof(float);
    cudaError_t e = cudaFuncSetAttribute(tree_attention_kernel<T, PIECES>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    GB_REQUIRE(e == cudaSuccess, "gb_tree_attention: %d bytes of shared memory refused: %s", smem, cudaGetErrorString(e));
    e = gb_launch(GB_PDL_ATTENTION, tree_attention_kernel<T, PIECES>, dim3(a.splits, tiles * a.nkv, num_seqs), dim3(TA_THREADS), smem, stream, a);
    GB_REQUIRE(e == cudaSuccess, "gb_tree_attention: launch failed: %s", cudaGetErrorString(e));
    return 0;
}

template <typename T>
static int ta_dispatch(const TreeArgs& a, int num_seqs, int max_rows, cudaStream_t stream) {
    const int tiles = gb_ceil_div((long long)max_rows * (a.nh / a.nkv), TA_ROWS);
    GB_REQUIRE((long long)tiles * a.nkv <= 65535, "gb_tree_attention: %d rows a request are too many for one launch", max_rows);
    int rc;
    if (a.hd <= 64) rc = ta_launch<T, 2>(a, num_seqs, tiles, stream);
    else if (a.hd <= 128) rc = ta_launch<T, 4>(a, num_seqs, tiles, stream);
    else rc = ta_launch<T, 8>(a, num_seqs, tiles, stream);
    return rc ? rc : gb_check_launch("gb_tree_attention");
}

// tree_attention_mma.cu, tree_attention_tc.cu
int gb_tree_attention_tc(const TreeArgs& a, const TreePlan& plan, int num_seqs, int max_rows, cudaStream_t stream);
int gb_tree_attention_mma(const TreeArgs& a, const TreePlan& plan, int num_seqs, int max_rows, cudaStream_t stream);
TreePlan tree_plan_mma(int num_seqs, int max_rows, int nh, int nkv, int hd, int max_context, int window, bool tc);

// Shares of a request's keys in this file's kernel, so that blocks fill the GPU, of 128 keys at least.
static int ta_splits(int num_seqs, int max_rows, int nh, int nkv, int max_context, int window) {
    const long long blocks = (long long)num_seqs * nkv * gb_ceil_div((long long)max_rows * (nh / nkv), TA_ROWS);
    const int reach = window > 0 && window + max_rows < max_context ? window + max_rows : max_context, most = reach <= 128 ? 1 : gb_ceil_div(reach, 128);
    const long long splits = 148ll * 3 / blocks;
    return splits > most ? most : splits < 1 ? 1 : (int)splits;
}

// Numbers (float32) of the scratch that a call needs; -1: more than there can be. kind as below.
GB_EXPORT int gb_tree_attention_floats(int kind, int n, int num_seqs, int max_rows, int nh, int nkv, int hd, int max_context, int window) {
    if (n <= 0 || num_seqs <= 0 || max_rows <= 0 || nkv <= 0 || nh % nkv) return 0;
    long long floats;
    if (kind >= 1) {
        floats = tree_plan_mma(num_seqs, max_rows, nh, nkv, hd, max_context, window, kind == 2).floats;
    } else {
        const int splits = ta_splits(num_seqs, max_rows, nh, nkv, max_context, window);
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
    TreeArgs a = {q, q_stride, out, out_stride, kcache, vcache, block_tables, max_pages, first_row, start_pos, positions, visible, words, n, nh, nkv, hd, page_size,
                  num_pages, scale, window, 1, parts, status};
    if (kind >= 1) {
        GB_REQUIRE(kind == 1 || (scale > 0.f && page_size >= 8 && page_size <= TREE_TC_KEYS && (uintptr_t)q % 16 == 0 && q_stride % 8 == 0 && (uintptr_t)out % 16 == 0 && out_stride % 8 == 0),
                   "gb_tree_attention: this scale, page size or alignment is not built for tcgen05");
        GB_REQUIRE(dtype == GB_BF16, "gb_tree_attention: the tensor cores' kernel takes bfloat16");
        const TreePlan plan = tree_plan_mma(num_seqs, max_rows, nh, nkv, hd, max_context, window, kind == 2);
        GB_REQUIRE(plan.floats == 0 || (parts != nullptr && (uintptr_t)parts % 16 == 0), "gb_tree_attention: the scratch is missing or not 16-byte aligned");
        return plan.tc ? gb_tree_attention_tc(a, plan, num_seqs, max_rows, stream) : gb_tree_attention_mma(a, plan, num_seqs, max_rows, stream);
    }
    a.splits = ta_splits(num_seqs, max_rows, nh, nkv, max_context, window);
    GB_REQUIRE(a.splits == 1 || parts != nullptr, "gb_tree_attention: the scratch is missing");
    const int rc = dtype == GB_F32 ? ta_dispatch<float>(a, num_seqs, max_rows, stream) : ta_dispatch<__nv_bfloat16>(a, num_seqs, max_rows, stream);
    if (rc || a.splits == 1) return rc;
    const unsigned blocks = (unsigned)(((size_t)n * nh + 3) / 4);
    const cudaError_t e = dtype == GB_F32 ? gb_launch(GB_PDL_ATTENTION, tree_merge_kernel<float>, dim3(blocks), dim3(128), 0, stream, a, num_seqs)
                                          : gb_launch(GB_PDL_ATTENTION, tree_merge_kernel<__nv_bfloat16>, dim3(blocks), dim3(128), 0, stream, a, num_seqs);
    GB_REQUIRE(e == cudaSuccess, "gb_tree_attention: launch failed: %s", cudaGetErrorString(e));
    return gb_check_launch("gb_tree_attention");
}
