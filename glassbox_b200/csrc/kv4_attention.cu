// Grouped-query attention over a cache in 4 bits (layout: kv4.cuh), one row at a time, the keys of a row cut into shares.
// A row at position p of its request sees keys max(0, p - window + 1) .. p, read through the request's block table. Scores, running maximum
// and sum and the output are float32; scores are in units of log 2, so that every exponential is a power of two.
//
// This file: the kernel that takes any row type and head size (float32 arithmetic throughout, one head of a row a block), and
// the merge of the shares. It is there to be right for float32 models, whose sums must not round a weight: a lane forms a key's score alone, one
// fused multiply-add a code, which bounds it (64 rows of 4/4 heads of 128 behind 2,048 keys: 90 us for 75 MB).
#include "kv4_attention.cuh"

constexpr int KV4R_WARPS = 4;
constexpr int KV4R_KEYS = 32;      // keys a warp takes at a time, one a lane

template <typename T>
__global__ void __launch_bounds__(KV4R_WARPS * 32) kv4_rows_kernel(const Kv4AttnArgs a) {
    __shared__ float qs[KV4_MAX_HD];
    __shared__ float ml[KV4R_WARPS][2];
    __shared__ float accs[KV4R_WARPS][KV4_MAX_HD];
    gb_pdl_launch_dependents();
    gb_pdl_wait();
    const int split = blockIdx.x, head = blockIdx.y, row = blockIdx.z;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, hd = a.hd, G = hd / KV4_GROUP, kvh = head / (a.nh / a.nkv);
    const T* q = (const T*)a.q + (size_t)row * a.q_stride + (size_t)head * hd;
    for (int i = threadIdx.x; i < hd; i += KV4R_WARPS * 32) qs[i] = gb_to_float(q[i]);
    __syncthreads();
    int pos = a.positions[row];
    if (pos >= 0 && pos / a.page_size >= a.max_pages) {   // a position the block table does not reach: reported, the row reads nothing
        if (threadIdx.x == 0) atomicOr(a.status, GB_STATUS_BAD_POSITION);
        pos = -1;
    }
    const int first = gb_first_key(pos, a.window);
    const int chunk0 = first / KV4R_KEYS, chunks = pos < 0 ? 0 : pos / KV4R_KEYS - chunk0 + 1;
    const int begin = chunk0 + kv4_share(chunks, split, gridDim.x), end = chunk0 + kv4_share(chunks, split + 1, gridDim.x);
    const int* table = a.block_tables + (size_t)a.row_seq[row] * a.max_pages;

    float m = KV4_NEG_BIG, l = 0.f, acc[KV4_MAX_HD / 32];
#pragma unroll
    for (int j = 0; j < KV4_MAX_HD / 32; ++j) acc[j] = 0.f;
    for (int c = begin + warp; c < end; c += KV4R_WARPS) {
        const int key = c * KV4R_KEYS + lane;
        const unsigned char* krow = nullptr;               // this lane's row of key codes; values lie at the same place of their pool
        long long at = -1;
        int r = 0;
        float s = -INFINITY;
        if (key >= first && key <= pos) {
            const long long page = table[key / a.page_size];
            const int off = key % a.page_size;
            if (page < 0 || page >= a.num_pages) {
                atomicOr(a.status, GB_STATUS_BAD_SLOT);
            } else {
                at = kv4_tile(page, kvh, off, a.nkv, a.page_size) * kv4_tile_bytes(hd);
                r = off % KV4_TILE;
                krow = a.kcache + at;
                s = 0.f;
                for (int g = 0; g < G; ++g) {
                    float d = 0.f;
#pragma unroll
                    for (int t = 0; t < 4; ++t) {
                        const unsigned w = *reinterpret_cast<const unsigned*>(krow + r * (hd / 2) + (t * G + g) * 4);
                        const float* x = qs + KV4_GROUP * g + 8 * t;
#pragma unroll
                        for (int j = 0; j < 8; ++j) d = fmaf(x[j], kv4_code(w, j), d);
                    }
                    s = fmaf(kv4_scale(krow, hd, r, g), d, s);
                }
                s *= a.scale;
            }
        }
        const float m_new = fmaxf(m, gb_warp_max(s)), p = at >= 0 ? exp2f(s - m_new) : 0.f, corr = exp2f(m - m_new);
        l = l * corr + gb_warp_sum(p);
#pragma unroll
        for (int j = 0; j < KV4_MAX_HD / 32; ++j) acc[j] *= corr;
        m = m_new;
        for (int k = 0; k < KV4R_KEYS; ++k) {
            const float pk = __shfl_sync(0xffffffffu, p, k);
            const long long where = __shfl_sync(0xffffffffu, at, k);
            const int rk = __shfl_sync(0xffffffffu, r, k);
            if (where < 0) continue;
            const unsigned char* tile = a.vcache + where;
#pragma unroll
            for (int j = 0; j < KV4_MAX_HD / 32; ++j) {
                if (j >= G) break;
                const unsigned w = *reinterpret_cast<const unsigned short*>(tile + rk * (hd / 2) + ((lane >> 2) * G + j) * 2);
                acc[j] = fmaf(pk, kv4_code(w, lane & 3) * kv4_scale(tile, hd, rk, j), acc[j]);
            }
        }
    }
    if (lane == 0) { ml[warp][0] = m; ml[warp][1] = l; }
#pragma unroll
    for (int j = 0; j < KV4_MAX_HD / 32; ++j)
        if (j < G) accs[warp][lane + 32 * j] = acc[j];
    __syncthreads();
    float most = KV4_NEG_BIG, sum = 0.f;
    for (int w = 0; w < KV4R_WARPS; ++w) most = fmaxf(most, ml[w][0]);
    for (int w = 0; w < KV4R_WARPS; ++w) sum += ml[w][1] * exp2f(ml[w][0] - most);
    float* part = a.parts + (((size_t)row * a.nh + head) * gridDim.x + split) * (hd + 2);
    for (int i = threadIdx.x; i < hd; i += KV4R_WARPS * 32) {
        float o = 0.f;
        for (int w = 0; w < KV4R_WARPS; ++w) o = fmaf(accs[w][i], exp2f(ml[w][0] - most), o);
        if (gridDim.x > 1) part[2 + i] = o;
        else ((T*)a.out)[(size_t)row * a.out_stride + (size_t)head * hd + i] = gb_from_float<T>(sum != 0.f ? o / sum : 0.f);
    }
    if (gridDim.x > 1 && threadIdx.x == 0) { part[0] = most; part[1] = sum; }
}

// The shares of a head's keys, (maximum, sum, output not yet divided) each, added up in their order: one block a row and head, a channel a thread.
template <typename T>
__global__ void kv4_merge_kernel(const float* __restrict__ parts, int shares, T* __restrict__ out, long long out_stride, int nh, int hd) {
    gb_pdl_launch_dependents();
    gb_pdl_wait();
    const int head = blockIdx.x, row = blockIdx.y, c = threadIdx.x;
    const float* p = parts + ((size_t)row * nh + head) * shares * (hd + 2);
    float m = KV4_NEG_BIG, l = 0.f, o = 0.f;
    for (int s = 0; s < shares; ++s) m = fmaxf(m, p[(size_t)s * (hd + 2)]);
    for (int s = 0; s < shares; ++s) {
        const float* share = p + (size_t)s * (hd + 2);
        const float f = exp2f(share[0] - m);
        l = fmaf(share[1], f, l);
        o = fmaf(share[2 + c], f, o);
    }
    out[(size_t)row * out_stride + (size_t)head * hd + c] = gb_from_float<T>(l != 0.f ? o / l : 0.f);
}

int kv4_merge(const Kv4AttnArgs& a, int dtype, int shares, cudaStream_t stream) {
    const dim3 grid(a.nh, a.n), block(a.hd);
    if (dtype == GB_F32)
        gb_launch(GB_PDL_ATTENTION, kv4_merge_kernel<float>, grid, block, 0, stream, a.parts, shares, (float*)a.out, a.out_stride, a.nh, a.hd);
    else
        gb_launch(GB_PDL_ATTENTION, kv4_merge_kernel<__nv_bfloat16>, grid, block, 0, stream, a.parts, shares, (__nv_bfloat16*)a.out, a.out_stride, a.nh, a.hd);
    return gb_check_launch("gb_kv4_attention_rows (merge)");
}

// Rows 0 .. n - 1, each at positions[r] of request row_seq[r]; a row of position < 0 comes out as zeros. parts (splits > 1): float32
// [n, nh, splits, hd + 2].
GB_EXPORT int gb_kv4_attention_rows(const void* q, long long q_stride, void* out, long long out_stride, int dtype, const void* kcache,
                                    const void* vcache, const int* block_tables, int max_pages, const int* row_seq, const int* positions,
                                    int n, int nh, int nkv, int hd, int page_size, long long num_pages, float scale, int window, int splits,
                                    float* parts, int* status, cudaStream_t stream) {
    KV4_REQUIRE_SIZES("gb_kv4_attention_rows")
    GB_REQUIRE(n >= 0 && nh > 0 && nh % nkv == 0 && max_pages > 0, "gb_kv4_attention_rows: bad sizes (rows %d, heads %d of %d, tables of %d pages)", n, nh, nkv, max_pages);
    GB_REQUIRE(dtype == GB_F32 || dtype == GB_BF16, "gb_kv4_attention_rows: unsupported dtype %d", dtype);
    GB_REQUIRE(splits >= 1 && (splits == 1 || parts != nullptr), "gb_kv4_attention_rows: %d shares need their scratch", splits);
    GB_REQUIRE((long long)max_pages * page_size < (1ll << 31) - 64, "gb_kv4_attention_rows: block tables of %d pages reach too far", max_pages);
    GB_REQUIRE(n <= 65535 && nh <= 65535, "gb_kv4_attention_rows: %d rows of %d heads are too many for one launch", n, nh);
    GB_REQUIRE(((uintptr_t)kcache | (uintptr_t)vcache) % 16 == 0, "gb_kv4_attention_rows: the cache must be 16-byte aligned");
    if (n == 0) return 0;
    Kv4AttnArgs a = {};
    a.q = q; a.q_stride = q_stride; a.out = out; a.out_stride = out_stride; a.kcache = (const unsigned char*)kcache;
    a.vcache = (const unsigned char*)vcache; a.block_tables = block_tables; a.max_pages = max_pages; a.row_seq = row_seq; a.positions = positions;
    a.n = n; a.nh = nh; a.nkv = nkv; a.hd = hd; a.page_size = page_size; a.num_pages = num_pages; a.scale = scale * KV4_LOG2E;
    a.window = window > 0 ? window : 0; a.parts = parts; a.status = status;
    const dim3 grid(splits, nh, n), block(KV4R_WARPS * 32);
    gb_launch(GB_PDL_ATTENTION, dtype == GB_F32 ? kv4_rows_kernel<float> : kv4_rows_kernel<__nv_bfloat16>, grid, block, 0, stream, a);
    if (int rc = gb_check_launch("gb_kv4_attention_rows")) return rc;
    return splits > 1 ? kv4_merge(a, dtype, splits, stream) : 0;
}
