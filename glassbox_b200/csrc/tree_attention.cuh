// Attention of a request's tree of drafted tokens over its paged cache: what the kernels for it share.
//
// Request s brings rows first_row[s] .. first_row[s + 1] - 1, its tree; row i of it lies in the cache at place start_pos[s] + i and at position
// positions[row] >= start_pos[s] of the text. With a window w, a row at position p sees of what lies before the tree the places above p - w, and
// of the tree the rows that its bits in `visible` name and whose positions are above p - w. The rows of a request times the query heads that share
// a key/value head are one list of R * G query rows, so that a tile of them reads each key and value once.
#pragma once
#include "common.cuh"

struct TreeArgs {
    const void* q;
    long long q_stride;
    void* out;
    long long out_stride;
    const void* kcache;
    const void* vcache;
    const int* block_tables;
    int max_pages, places;   // (places: of the pages' tokens)
    const int* first_row;
    const int* start_pos;
    const int* positions;
    const int* visible;      // [n, words], 32 rows of the tree a word
    int words;
    int n, max_rows, nh, nkv, hd, page_size;
    long long num_pages;
    float scale;
    int window;              // 0: none
    int splits;              // (tree_attention.cu)
    float* parts;
    int* status;
};

// How a batch is laid out over the GPU.
struct TreePlan {
    int rows = 0;            // query rows of an item
    int cluster = 0;         // blocks that share an item's keys, a cluster; 0: all items' keys are cut evenly among `blocks`
    int blocks = 0;
    bool tc = false;         // by tree_attention_tc.cu, in `blocks` blocks
    bool same = false;       // its items have at most 128 query rows
    long long floats = 0;    // of scratch
};

// Rows of a request; -1: they lie outside the batch, or are more than was said, for which neither grid nor scratch is made.
__device__ __forceinline__ int tree_rows(const TreeArgs& a, int seq) {
    const int row0 = a.first_row[seq], rows = a.first_row[seq + 1] - row0;
    return row0 < 0 || rows < 0 || row0 > a.n - rows || rows > a.max_rows ? -1 : rows;
}

// A request of the step. rows 0: nothing to do.
struct TreeSeq {
    int row0, rows, start, key_lo, length;
    const int* table;
    __device__ __forceinline__ TreeSeq(const TreeArgs& a, int seq) {
        row0 = a.first_row[seq];
        rows = tree_rows(a, seq);
        start = a.start_pos[seq];
        table = a.block_tables + (size_t)seq * a.max_pages;
        if (rows < 0) {                                   // (reported, nothing is read or written)
            atomicOr(a.status, GB_STATUS_BAD_SLOT);
            rows = 0;
        } else if (rows > 0 && start > a.places - rows) { // (nor where the tables do not reach)
            atomicOr(a.status, GB_STATUS_BAD_POSITION);
            rows = 0;
        }
        length = start + rows;
        key_lo = a.window > 0 ? max(0, start - a.window + 1) : 0;
    }
    // Tiles of `keys` keys (a multiple of them behind place 0) that hold what any row sees.
    __device__ __forceinline__ int tiles(int keys) const { return rows > 0 && start >= 0 ? (length + keys - 1) / keys - key_lo / keys : 0; }
    // The page of a place, -1 where there is none.
    __device__ __forceinline__ int page(const TreeArgs& a, int index) const {
        const int p = index < a.max_pages ? table[index] : -1;
        return p >= 0 && p < a.num_pages ? p : -1;
    }
    // Whether the row (of the batch) at position `pos` sees the key at a place.
    __device__ __forceinline__ bool sees(const TreeArgs& a, int row, int pos, int key) const {
        if (key >= length) return false;
        if (key < start) return a.window <= 0 || pos - key < a.window;
        const int d = key - start;
        if ((d >> 5) >= a.words || !((unsigned)a.visible[(size_t)row * a.words + (d >> 5)] >> (d & 31) & 1u)) return false;
        return a.window <= 0 || pos - a.positions[row0 + d] < a.window;
    }
};

// Of the 32 rows of the tree from d0 on (negative: keys before the tree, all seen), those that a row of the batch sees. `only`: its
// bits, where they are one word.
__device__ __forceinline__ unsigned tree_bits(const TreeArgs& a, int rows, int row, int d0, unsigned only) {
    if (d0 <= -32) return 0xffffffffu;
    if (row < 0) return 0u;
    const unsigned* bits = reinterpret_cast<const unsigned*>(a.visible) + (size_t)row * a.words;
    unsigned v;
    if (d0 < 0) {
        v = ((1u << -d0) - 1u) | ((a.words == 1 ? only : bits[0]) << -d0);
    } else if (a.words == 1) {
        v = d0 < 32 ? only >> d0 : 0u;
    } else {
        const int w = d0 >> 5, sh = d0 & 31;
        v = w < a.words ? bits[w] >> sh : 0u;
        if (sh && w + 1 < a.words) v |= bits[w + 1] << (32 - sh);
    }
    const int left = rows - d0;
    return left >= 32 ? v : left <= 0 ? 0u : v & ((1u << left) - 1u);
}

__device__ __forceinline__ unsigned tree_bits(const TreeArgs& a, int rows, int row, int d0) {
    return tree_bits(a, rows, row, d0, row >= 0 && a.words == 1 && d0 > -32 ? (unsigned)a.visible[row] : 0u);
}

constexpr int TREE_TC_KEYS = 128, TREE_TC_ROWS = 128;      // keys of a tile and rows of a unit of tree_attention_tc.cu
constexpr int TREE_LEAST_SHARE = 4;      // tiles of keys of a block, where there are enough

// All items' tiles of keys in one row, request by request, key/value head by head, `rows` query rows at a time, cut evenly among the blocks. Every warp works
// it out for itself from the requests' lengths, which only the device knows.
struct TreeCut {
    const TreeArgs& a;
    int num_seqs, rows, keys;
    long long total, share;
    int seq;                 // a request, the tiles and items before it
    long long tile0, item0, tiles_here;
    __device__ __forceinline__ void of(int s, long long& tiles, long long& items) const {
        tiles = items = 0;
        if (s >= num_seqs) return;
        const int n = tree_rows(a, s), start = a.start_pos[s];
        if (n <= 0 || start < 0 || start > a.places - n) return;
        const int low = a.window > 0 ? max(0, start - a.window + 1) : 0;
        items = (long long)a.nkv * ((n * (a.nh / a.nkv) + rows - 1) / rows);
        tiles = items * ((start + n + keys - 1) / keys - low / keys);
    }
    __device__ __forceinline__ static long long scan(long long v) {
        const int lane = threadIdx.x & 31;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long up = __shfl_up_sync(0xffffffffu, v, o);
            if (lane >= o) v += up;
        }
        return v;
    }
    __device__ __forceinline__ TreeCut(const TreeArgs& a, int num_seqs, int rows, int keys, int blocks, int least)
        : a(a), num_seqs(num_seqs), rows(rows), keys(keys) {
        long long sum = 0;
        for (int s0 = 0; s0 < num_seqs; s0 += 32) {
            long long t, i;
            of(s0 + (threadIdx.x & 31), t, i);
            sum += t;
        }
        total = __shfl_sync(0xffffffffu, scan(sum), 31);
        share = (total + blocks - 1) / blocks;
        if (share < least) share = least;
    }
    // The request that holds tile `at`.
    __device__ __forceinline__ void seek(long long at) { find(at, -1); }
    __device__ __forceinline__ void seek_seq(int s) { find(-1, s); }
    __device__ __forceinline__ void find(long long at, int want) {
        const int lane = threadIdx.x & 31;
        long long tiles_before = 0, items_before = 0;
        for (int s0 = 0; s0 < num_seqs; s0 += 32) {
            long long t, i;
            of(s0 + lane, t, i);
            const long long ts = scan(t), is = scan(i);
            const unsigned hit = __ballot_sync(0xffffffffu, want >= 0 ? s0 + lane == want : t > 0 && tiles_before + ts > at);
            if (hit) {
                const int l = __ffs(hit) - 1;
                seq = s0 + l;
                tiles_here = __shfl_sync(0xffffffffu, t, l);
                tile0 = tiles_before + __shfl_sync(0xffffffffu, ts, l) - tiles_here;
                item0 = items_before + __shfl_sync(0xffffffffu, is - i, l);
                return;
            }
            tiles_before += __shfl_sync(0xffffffffu, ts, 31);
            items_before += __shfl_sync(0xffffffffu, is, 31);
        }
        seq = -1;
        tile0 = item0 = tiles_here = 0;
    }
    // On to the request that holds tile `at`, which comes later.
    __device__ __forceinline__ void reach(long long at) {
        while (at >= tile0 + tiles_here) {
            long long t, i;
            of(seq, t, i);
            tile0 += tiles_here;
            item0 += i;
            ++seq;
            of(seq, tiles_here, i);
        }
    }
};
