// What the attention kernels over a cache in 4 bits share.
#pragma once
#include "kv4.cuh"

constexpr float KV4_NEG_BIG = -1.0e30f;             // (finite: differences of two of them are numbers)
constexpr float KV4_LOG2E = 1.4426950408889634f;

struct Kv4AttnArgs {
    const void* q;
    long long q_stride;
    void* out;
    long long out_stride;
    const unsigned char* kcache;
    const unsigned char* vcache;
    const int* block_tables;
    int max_pages;
    const int* row_seq;
    const int* positions;
    int n, nh, nkv, hd, page_size;
    long long num_pages;
    float scale;                 // of the scores, times log2(e)
    int window;                  // keys that a row sees at most; 0: all
    float* parts;                // [n, nh, shares, hd + 2]: maximum, sum, output not yet divided
    int* status;
};

// Where share `s` of `shares` begins among `count` things.
__device__ __forceinline__ int kv4_share(int count, int s, int shares) { return (int)((long long)count * s / shares); }

// Adds up a.parts into a.out (kv4_attention.cu).
int kv4_merge(const Kv4AttnArgs& a, int dtype, int shares, cudaStream_t stream);
