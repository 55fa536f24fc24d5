// Keeping what is accepted of a request's tree of drafted tokens: the keys and values of its kept rows move, in every layer, from the places where the step
// wrote them (start + path[j]) to the places directly behind what the cache held before (start + j).
//
// path ascends, so j <= path[j], and a place that is written has been read before by whoever goes through j in order: a thread has one piece of a head's rows
// and takes the moves eight at a time, all loads before the first store. What bounds it is the trip to memory for pieces of 16 bytes, few of them.
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
__global__ void __launch_bounds__(KR_THREADS) keep_rows_kernel(const KeepArgs a) {
    __shared__ long long from[KR_MAX_ROWS], to[KR_MAX_ROWS];      // places of the pool (page * page_size + offset)
    __shared__ int moves, wrong;
    const int seq = blockIdx.x, which = blockIdx.y & 1, tid = threadIdx.x;
    const long long layer = blockIdx.y >> 1;
    gb_pdl_launch_dependents();
    gb_pdl_wait();
    const int row0 = a.first_row[seq], rows = a.first_row[seq + 1] - row0, start = a.start_pos[seq], kept = a.accepted[seq];
    if (start < 0 || rows <= 0 || kept <= 0) return;
    if (tid == 0) { moves = 0; wrong = 0; }
    __syncthreads();
    if (row0 < 0 || row0 > a.n - rows || kept > rows || rows > KR_MAX_ROWS) {
        if (tid == 0) atomicOr(a.status, GB_STATUS_BAD_POSITION);
        return;
    }
    const int* table = a.block_tables + (size_t)seq * a.max_pages;
    auto place = [&](int at) -> long long {
        const int index = at / a.page_size;
        const int page = index < a.max_pages ? table[index] : -1;
        if (page < 0 || page >= a.num_pages) return -1;
        return (long long)page * a.page_size + at % a.page_size;
    };
    for (int j = tid; j < kept; j += KR_THREADS) {
        const int r = a.path[row0 + j];
        long long src = -1, dst = -1;
        if (r >= j && r < rows) {
            src = place(start + r);
            dst = place(start + j);
        }
        if (src < 0 || dst < 0) wrong = 1;
        from[j] = src;
        to[j] = dst;
        if (r != j) atomicMax(&moves, j + 1);         // (rows before the first that moves are skipped below by their own places)
    }
    __syncthreads();
    if (wrong) {                                      // a path that does not ascend in the tree, or a page that is missing: nothing moves
        if (tid == 0) atomicOr(a.status, GB_STATUS_BAD_SLOT);
        return;
    }
    const int pieces = a.row_bytes[which] / (int)sizeof(V), each = a.page_size * pieces;
    V* pool = reinterpret_cast<V*>(a.pool[which]) + layer * a.num_pages * a.heads * each;
    for (int i = tid + blockIdx.z * KR_THREADS; i < a.heads * pieces; i += KR_THREADS * gridDim.z) {
        const int head = i / pieces, c = i % pieces;
        auto cell = [&](long long p) { return pool + ((p / a.page_size * a.heads + head) * a.page_size + p % a.page_size) * pieces + c; };
        for (int j0 = 0; j0 < moves; j0 += KR_FLY) {
            V v[KR_FLY];
#pragma unroll
            for (int u = 0; u < KR_FLY; ++u)
                if (j0 + u < moves && from[j0 + u] != to[j0 + u]) v[u] = *cell(from[j0 + u]);
#pragma unroll
            for (int u = 0; u < KR_FLY; ++u)
                if (j0 + u < moves && from[j0 + u] != to[j0 + u]) *cell(to[j0 + u]) = v[u];
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
    const dim3 grid(num_seqs, 2 * layers, gb_ceil_div((long long)heads * (most / size), KR_THREADS));
    GB_REQUIRE(grid.z <= 65535, "gb_keep_rows: rows too long");
    const auto kernel = size == 16 ? keep_rows_kernel<uint4> : size == 8 ? keep_rows_kernel<uint2> : size == 4 ? keep_rows_kernel<uint32_t> : keep_rows_kernel<uint16_t>;
    const cudaError_t e = gb_launch(GB_PDL_ELEMENTWISE, kernel, grid, dim3(KR_THREADS), 0, stream, a);
    GB_REQUIRE(e == cudaSuccess, "gb_keep_rows: launch failed: %s", cudaGetErrorString(e));
    return gb_check_launch("gb_keep_rows");
}
