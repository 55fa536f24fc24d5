// Keeping what is accepted of a request's tree of drafted tokens: the keys and values of its kept rows move, in every layer, from the places where the step
// wrote them (start + path[j]) to the places directly behind what the cache held before (start + j).
//
// path ascends, so j <= path[j], and a place that is written has been read before by whoever goes through j in order: a thread has one piece of a head's rows
// and takes the moves eight at a time, all loads before the first store. A block lists a request's moves once and goes through several layers' keys and values.
// What bounds it: the trips to memory before the first piece moves (who moves, whereto, the page, the piece), and pieces of 16 bytes: 1 request, 30 layers of 3 heads
// of 64, 4.2 us; 64 requests, 24 layers of 32 heads of 64 (100 MB read and written) 24.7 us, 4.1 TB/s.
#include "common.cuh"

constexpr int KR_THREADS = 256, KR_FLY = 8, KR_MAX_ROWS = 1024;

struct KeepArgs {
    unsigned char* pool[2];
    int row_bytes[2];            // of a place and head, of keys and of values
    int heads, page_size, max_pages;
    long long num_pages;
    const int* block_tables;
    const int* first_row;
    const int* start_pos;
    const int* path;
    const int* accepted;
    int n;
    int* status;
};

template <typename V>
__global__ void __launch_bounds__(KR_THREADS) keep_rows_kernel(const KeepArgs a, int pools, int per) {
    __shared__ long long from[KR_MAX_ROWS], to[KR_MAX_ROWS];      // rows of head 0 of the pool
    __shared__ int moves, wrong;
    const int seq = blockIdx.x, tid = threadIdx.x, lane = tid & 31;
    gb_pdl_launch_dependents();
    gb_pdl_wait();
    const int row0 = a.first_row[seq], rows = a.first_row[seq + 1] - row0, start = a.start_pos[seq], kept = a.accepted[seq];
    if (start < 0 || rows <= 0 || kept <= 0) return;
    if (row0 < 0 || row0 > a.n - rows || kept > rows || rows > KR_MAX_ROWS) {
        if (tid == 0) atomicOr(a.status, GB_STATUS_BAD_POSITION);
        return;
    }
    if (tid < 32) {
        const int* table = a.block_tables + (size_t)seq * a.max_pages;
        auto place = [&](int from, int rows) -> long long {
            const unsigned at = (unsigned)from + (unsigned)rows, index = at / (unsigned)a.page_size;      // (may pass 2^31)
            const int page = index < (unsigned)a.max_pages ? table[index] : -1;
            if (page < 0 || page >= a.num_pages) return -1;
            return (long long)page * a.heads * a.page_size + at % (unsigned)a.page_size;
        };
        int count = 0;
        bool bad = false;
        for (int j0 = 0; j0 < kept; j0 += 32) {
            const int j = j0 + lane, r = j < kept ? a.path[row0 + j] : j;
            long long src = 0, dst = 0;
            if (r != j) {
                if (r > j && r < rows) {
                    src = place(start, r);
                    dst = place(start, j);
                }
                bad = bad || src == dst || src < 0 || dst < 0;      // (a path that leaves its tree or does not ascend, or a page that is missing)
            }
            const unsigned who = __ballot_sync(0xffffffffu, r != j);
            if (r != j) {
                const int at = count + __popc(who & ((1u << lane) - 1u));
                from[at] = src;
                to[at] = dst;
            }
            count += __popc(who);
        }
        bad = __any_sync(0xffffffffu, bad);
        if (lane == 0) { moves = count; wrong = bad; }
    }
    __syncthreads();
    if (wrong) {                                      // nothing moves
        if (tid == 0) atomicOr(a.status, GB_STATUS_BAD_SLOT);
        return;
    }
    if (moves == 0) return;
    for (int p = blockIdx.y * per; p < min(pools, (int)(blockIdx.y + 1) * per); ++p) {
        const int which = p & 1, pieces = a.row_bytes[which] / (int)sizeof(V);
        V* pool = reinterpret_cast<V*>(a.pool[which]) + (long long)(p >> 1) * a.num_pages * a.heads * a.page_size * pieces;
        for (int i = tid + blockIdx.z * KR_THREADS; i < a.heads * pieces; i += KR_THREADS * gridDim.z) {
            const int head = i / pieces, c = i % pieces;
            V* mine = pool + (long long)head * a.page_size * pieces + c;
            for (int j0 = 0; j0 < moves; j0 += KR_FLY) {
                V v[KR_FLY];
#pragma unroll
                for (int u = 0; u < KR_FLY; ++u)
                    if (j0 + u < moves) v[u] = mine[from[j0 + u] * pieces];
#pragma unroll
                for (int u = 0; u < KR_FLY; ++u)
                    if (j0 + u < moves) mine[to[j0 + u] * pieces] = v[u];
            }
        }
    }
}

// Pools [layers, num_pages, heads, page_size, row bytes], contiguous. Row j of request s that is kept (j < accepted[s]) is row path[first_row[s] + j] of its tree.
GB_EXPORT int gb_keep_rows(void* kpool, void* vpool, int krow_bytes, int vrow_bytes, int layers, long long num_pages, int heads, int page_size,
                           const int* block_tables, int max_pages, const int* first_row, const int* start_pos, const int* path, const int* accepted, int n,
                           int num_seqs, int* status, cudaStream_t stream) {
    GB_REQUIRE(layers > 0 && layers <= 32767 && num_pages > 0 && heads > 0 && page_size > 0 && max_pages > 0 && num_seqs >= 0 && n >= 0, "gb_keep_rows: bad sizes");
    GB_REQUIRE(krow_bytes > 0 && vrow_bytes > 0, "gb_keep_rows: bad row sizes");
    GB_REQUIRE((long long)max_pages * page_size < (1ll << 31) - 4096, "gb_keep_rows: the block tables reach too far");
    if (num_seqs == 0 || n == 0) return 0;
    GB_REQUIRE(kpool && vpool && block_tables && first_row && start_pos && path && accepted && status, "gb_keep_rows: a tensor is missing");
    KeepArgs a = {{(unsigned char*)kpool, (unsigned char*)vpool}, {krow_bytes, vrow_bytes}, heads, page_size, max_pages, num_pages, block_tables, first_row, start_pos,
                  path, accepted, n, status};
    int size = 16;
    while (size > 1 && (krow_bytes % size || vrow_bytes % size || (uintptr_t)kpool % size || (uintptr_t)vpool % size)) size /= 2;
    GB_REQUIRE(size >= 2, "gb_keep_rows: rows of %d and %d bytes at an odd address", krow_bytes, vrow_bytes);
    const int most = krow_bytes > vrow_bytes ? krow_bytes : vrow_bytes;
    // as many layers' keys or values a block as leave eight blocks a multiprocessor: 64 requests of 30 layers of 3 heads of 64, one / two / four / 48 a block
    // 18.5 / 12.4 / 10.3 / 28.8 us; 8 requests of 24 layers of 32 heads of 64, one / four / eight 6.2 / 8.3 / 10.3
    const unsigned parts = gb_ceil_div((long long)heads * (most / size), KR_THREADS);
    GB_REQUIRE(parts <= 65535, "gb_keep_rows: rows too long");
    long long per = (long long)num_seqs * parts * 2 * layers / (8 * 148);
    per = per < 1 ? 1 : per > 2 * layers ? 2 * layers : per;
    const dim3 grid(num_seqs, gb_ceil_div(2 * layers, per), parts);
    const auto kernel = size == 16 ? keep_rows_kernel<uint4> : size == 8 ? keep_rows_kernel<uint2> : size == 4 ? keep_rows_kernel<uint32_t> : keep_rows_kernel<uint16_t>;
    const cudaError_t e = gb_launch(GB_PDL_ELEMENTWISE, kernel, grid, dim3(KR_THREADS), 0, stream, a, 2 * layers, (int)per);
    GB_REQUIRE(e == cudaSuccess, "gb_keep_rows: launch failed: %s", cudaGetErrorString(e));
    return gb_check_launch("gb_keep_rows");
}
