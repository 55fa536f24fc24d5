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
    int max_pages;
    const int* first_row;
    const int* start_pos;
    const int* positions;
    const int* visible;      // [n, words], 32 rows of the tree a word
    int words;
    int n, nh, nkv, hd, page_size;
    long long num_pages;
    float scale;
    int window;              // 0: none
    int splits;
    float* parts;            // splits > 1: [splits, n, nh, hd] unnormalised outputs, then [splits, n, nh, 2] maxima (of scores times scale, base 2) and sums
    int* status;
};

// A request of the step. rows 0: nothing to do.
struct TreeSeq {
    int row0, rows, start, key_lo, length;
    const int* table;
    __device__ __forceinline__ TreeSeq(const TreeArgs& a, int seq) {
        row0 = a.first_row[seq];
        rows = a.first_row[seq + 1] - row0;
        start = a.start_pos[seq];
        table = a.block_tables + (size_t)seq * a.max_pages;
        if (row0 < 0 || rows < 0 || row0 > a.n - rows) {          // (rows outside the batch: reported, nothing is read or written)
            atomicOr(a.status, GB_STATUS_BAD_SLOT);
            rows = 0;
        }
        length = start + rows;
        key_lo = a.window > 0 ? max(0, start - a.window + 1) : 0;
    }
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
