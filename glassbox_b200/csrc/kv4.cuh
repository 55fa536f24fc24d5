// A cache of keys and values in 4 bits: the layout that its kernels share.
//
// 32 neighbouring channels of a token and head are a group. With m its number of the largest magnitude (the positive one of two) the
// group's scale is d = -m / 8 rounded to five significant bits, and a number x is held as s, the whole number from -8 to 7 nearest to x / d: it
// stands for s d. Five bits of d and three of s (-8 needs one) make a product that bfloat16 holds exactly, so that what reads the cache
// directly and what unpacks it into bfloat16 pages first work with the same numbers. The largest number lands on -8 whatever its
// sign, so all sixteen codes are in use; the far end of the other sign is cut off at 7. A group with a number that is not finite gets
// the scale NaN; one whose numbers are all below 2^-117 the scale zero (nothing near the subnormal numbers is divided).
//
// A page of a head is a run of tiles of 16 tokens; a tile (9 hd bytes) is what one asynchronous copy brings: 16 rows of hd / 2 bytes of
// codes s + 8 (two in a byte, the first in the low half), then 16 rows of hd / 32 scales in bfloat16. Channels lie in a row of codes
// in the order in which the fragments of mma.m16n8k16 want them (G = hd / 32 groups):
//   keys:   nibble ((c % 32) / 8 * G + c / 32) * 8 + c % 8: the eight channels of a group that a lane of a quad holds are a word,
//           and a quad's lane finds its words of all groups side by side;
//   values: nibble ((c % 32) / 4 * G + c / 32) * 4 + c % 4: the four channels of a group that one of eight lanes holds are a half word,
//           a lane's of all groups side by side.
#pragma once
#include "common.cuh"

constexpr int KV4_TILE = 16;       // tokens of a tile
constexpr int KV4_GROUP = 32;      // channels that share a scale
constexpr int KV4_MAX_HD = 256;

__host__ __device__ __forceinline__ constexpr int kv4_tile_bytes(int hd) { return 9 * hd; }

// Quotients by a divisor that a launch fixes: the high half of the product with 2^32 / d rounded up, exact while x d < 2^32.
struct Kv4Div {
    unsigned d, m;
    __host__ Kv4Div(int divisor = 1) : d((unsigned)divisor), m(divisor > 1 ? (unsigned)(((1ull << 32) + divisor - 1) / divisor) : 0u) {}
    __device__ __forceinline__ int of(int x) const { return d == 1u ? x : (int)__umulhi((unsigned)x, m); }
};

// The tile of token `off` of a page of kv head `head`, counted over the whole pool.
__device__ __forceinline__ long long kv4_tile(long long page, int head, int off, int nkv, int page_size) {
    return (page * nkv + head) * (page_size / KV4_TILE) + off / KV4_TILE;
}

__device__ __forceinline__ float kv4_scale(const unsigned char* tile, int hd, int row, int group) {
    const unsigned short s = *reinterpret_cast<const unsigned short*>(tile + 8 * hd + (row * (hd / KV4_GROUP) + group) * 2);
    return __uint_as_float((unsigned)s << 16);
}

// code j of a word (or half word) as a number
__device__ __forceinline__ float kv4_code(unsigned word, int j) { return (float)((int)((word >> (4 * j)) & 15u) - 8); }

#define KV4_REQUIRE_SIZES(what)                                                                                                              \
    GB_REQUIRE(nkv > 0 && hd > 0 && hd % KV4_GROUP == 0 && hd <= KV4_MAX_HD, what ": head size %d must be a multiple of 32 up to 256", hd); \
    GB_REQUIRE(page_size > 0 && page_size % KV4_TILE == 0, what ": page size %d must be a multiple of 16", page_size);                       \
    GB_REQUIRE(num_pages > 0 && num_pages * page_size < (1ll << 31) && num_pages * page_size / KV4_TILE * nkv < (1ll << 31),               \
               what ": a pool of %lld pages of %d tokens and %d heads is too large", (long long)num_pages, page_size, nkv);
