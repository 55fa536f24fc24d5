// Writing a cache in 4 bits and reading it back (layout: kv4.cuh). Three kernels:
//   kv4_write   rotates the queries and keys of a step's rows, rounds keys and values to 4 bits and stores them in their pages;
//   kv4_read    what the cache holds for given slots, as numbers;
//   kv4_expand  the pages that a step's requests see, as pages of bfloat16 or float32 that the prompt kernels read.
// What they cannot do without is bytes: a row of a wide layout (32/8 heads of 128, bfloat16) brings 12 KB in, 8 KB of queries out and 1.1 KB of
// cache out.
//
// The rounding: m's bits less 3 in the exponent, rounded to four bits after the leading one, are |d|. A quotient y / d is the product with the
// reciprocal and one correction by the remainder (exact in a fused multiply-add), so that a number half way between two codes is told as such:
// with bfloat16 values that is one in dozens, and ties go to the even code. A rotated key is a float32 product off by some 2^-23; where that
// could change a code or the scale (one group in some 10^4) the group is held once more from two float32 a number, so that what
// is stored is what the exact rotation gives wherever that is not nearer than some 2^-46 of a pair's size to a border.
#include "kv4.cuh"

#include <type_traits>

// Measured (bfloat16, 32/8 heads of 128 of which 64 channels turn, 8,000 rows written and read back, 217 MB): 62 us; without the queries 40, without
// keys 46, without values 53. Neither instructions (58 % of the issue slots) nor memory (32 % of its rate) fill it: what bounds it is a block's one
// round of loads and the chain of maxima and codes behind them. A thread has two loads or more under way: with one
// piece of a query a thread and keys and values read back apart it took 84, with two pieces of one head 67. 64 / 256 threads a block took 117 / 87
// where 128 took 84; 40 registers (12 blocks a multiprocessor) take 72 where 56 take 62.
constexpr int KV4_THREADS = 128;

template <typename T, int N> struct Kv4Load;      // N neighbouring numbers as float32 (N * sizeof(T) bytes, aligned to 16 or to all of them)
template <> struct Kv4Load<float, 8> {
    static __device__ __forceinline__ void load(const float* p, float (&f)[8]) {
        const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
        f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w; f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
    }
    static __device__ __forceinline__ void store(float* p, const float (&f)[8]) {
        *reinterpret_cast<float4*>(p) = make_float4(f[0], f[1], f[2], f[3]);
        *reinterpret_cast<float4*>(p + 4) = make_float4(f[4], f[5], f[6], f[7]);
    }
};
template <> struct Kv4Load<float, 4> {
    static __device__ __forceinline__ void load(const float* p, float (&f)[4]) {
        const float4 a = *reinterpret_cast<const float4*>(p);
        f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
    }
    static __device__ __forceinline__ void store(float* p, const float (&f)[4]) { *reinterpret_cast<float4*>(p) = make_float4(f[0], f[1], f[2], f[3]); }
};
__device__ __forceinline__ uint32_t kv4_pair(float lo, float hi) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}
template <> struct Kv4Load<__nv_bfloat16, 8> {
    static __device__ __forceinline__ void load(const __nv_bfloat16* p, float (&f)[8]) {
        const uint4 a = *reinterpret_cast<const uint4*>(p);
        const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            f[2 * i] = __uint_as_float(w[i] << 16);
            f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
    }
    static __device__ __forceinline__ void store(__nv_bfloat16* p, const float (&f)[8]) {
        *reinterpret_cast<uint4*>(p) = make_uint4(kv4_pair(f[0], f[1]), kv4_pair(f[2], f[3]), kv4_pair(f[4], f[5]), kv4_pair(f[6], f[7]));
    }
};
template <> struct Kv4Load<__nv_bfloat16, 4> {
    static __device__ __forceinline__ void load(const __nv_bfloat16* p, float (&f)[4]) {
        const uint2 a = *reinterpret_cast<const uint2*>(p);
        f[0] = __uint_as_float(a.x << 16); f[1] = __uint_as_float(a.x & 0xffff0000u);
        f[2] = __uint_as_float(a.y << 16); f[3] = __uint_as_float(a.y & 0xffff0000u);
    }
    static __device__ __forceinline__ void store(__nv_bfloat16* p, const float (&f)[4]) {
        *reinterpret_cast<uint2*>(p) = make_uint2(kv4_pair(f[0], f[1]), kv4_pair(f[2], f[3]));
    }
};

// WIDE: rows are aligned for 16-byte loads; otherwise number by number.
template <typename T, int N, bool WIDE>
__device__ __forceinline__ void kv4_load(const T* p, float (&f)[N]) {
    if (WIDE) {
        Kv4Load<T, N>::load(p, f);
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) f[i] = gb_to_float(p[i]);
    }
}
template <typename T, int N, bool WIDE>
__device__ __forceinline__ void kv4_store(T* p, const float (&f)[N]) {
    if (WIDE) {
        Kv4Load<T, N>::store(p, f);
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) p[i] = gb_from_float<T>(f[i]);
    }
}

// N numbers in 16-byte pieces, asked for and looked at later.
template <typename T, int N> struct Kv4Asked {
    static constexpr int WORDS = N * (int)sizeof(T) / 4;
    uint32_t w[WORDS];
    __device__ __forceinline__ void ask(const T* p) {
#pragma unroll
        for (int i = 0; i < WORDS; i += 4) {
            const uint4 v = *reinterpret_cast<const uint4*>(p + i * 4 / (int)sizeof(T));
            w[i] = v.x; w[i + 1] = v.y; w[i + 2] = v.z; w[i + 3] = v.w;
        }
    }
    __device__ __forceinline__ void get(float (&f)[N]) const {
#pragma unroll
        for (int i = 0; i < N; ++i)
            f[i] = sizeof(T) == 4 ? __uint_as_float(w[i % WORDS]) : __uint_as_float(i & 1 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
    }
};

__device__ __forceinline__ float kv4_max_nan(float a, float b) {           // NaN where one of them is
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float kv4_min_nan(float a, float b) {
    float r;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float kv4_max_nan(float a, float b, float c) {
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
__device__ __forceinline__ float kv4_min_nan(float a, float b, float c) {
    float r;
    asm("min.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
// The largest and the smallest of N numbers of this thread.
template <int N>
__device__ __forceinline__ void kv4_ends(const float (&y)[N], float& high, float& low) {
    high = kv4_max_nan(y[0], y[1]);
    low = kv4_min_nan(y[0], y[1]);
#pragma unroll
    for (int i = 2; i < N; i += 2) {
        high = kv4_max_nan(high, y[i], y[i + 1]);
        low = kv4_min_nan(low, y[i], y[i + 1]);
    }
}

// Bits of a magnitude's scale: an eighth of it, four bits after the leading one, ties to even.
__device__ __forceinline__ unsigned kv4_five(unsigned size) {
    const unsigned d = size - (3u << 23);
    return (d + 0x3ffffu + ((d >> 19) & 1u)) & 0xfff80000u;
}

// The scale of a group from its ends, as float32: zero, NaN, or a number of five significant bits.
__device__ __forceinline__ float kv4_make_scale(float high, float low) {
    const float m = high >= -low ? high : low, size = fabsf(m);
    if (!(fmaxf(high, -low) <= FLT_MAX && high == high && low == low)) return __uint_as_float(0x7fc00000u);
    if (size < 6.018531076210112e-36f) return 0.f;                         // 2^-117
    return __uint_as_float(kv4_five(__float_as_uint(size)) | (m > 0.f ? 0x80000000u : 0u));
}

// Codes s + 8 of N numbers, N nibbles from the low end on: the quotient y / d (to within a rounding; exactly half way where it is), limited, plus
// 1.5 2^23 + 8, which rounds it and leaves the code in the lowest bits; the words of bits are added up as digits of base 16 with what the
// others of their bits come to taken off at the end. near: the farthest that a quotient lies from its code.
template <int N>
__device__ __forceinline__ unsigned kv4_codes(const float (&y)[N], float d, float& near) {
    near = 0.f;
    if (!(fabsf(d) > 0.f)) return 0x88888888u;                             // nothing, or NaN: s = 0
    constexpr float WHOLE = 12582920.f;
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(d));
    unsigned w = 0x100000000ull - 0x3f400000u;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        float q = y[i] * r;
        q = fminf(fmaxf(fmaf(fmaf(-q, d, y[i]), r, q), -8.f), 7.f);
        const float t = q + WHOLE;
        near = fmaxf(near, fabsf(q - (t - WHOLE)));
        w += __float_as_uint(t) << (4 * i);
    }
    return w;
}

// The same for numbers that are bfloat16. 2 y / d has a denominator of at most 31 (d's five bits) behind the digits of y's eight, so a quotient that
// is not half way between two codes is 2^-9 off at least, and one rounded to 2^-13 by a first sum (the product with the reciprocal is off by less than
// 2^-19) is half way where y / d is. The largest magnitude has the sign of -8, so that only 7 limits; its 8.26 at most rounds to 8.
template <int N>
__device__ __forceinline__ unsigned kv4_codes_bf16(const float (&y)[N], float d) {
    if (!(fabsf(d) > 0.f)) return 0x88888888u;
    constexpr float WHOLE = 12582920.f, FINE = 1536.f;
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(d));
    unsigned w = 0x100000000ull - 0x3f400000u;
#pragma unroll
    for (int i = 0; i < N; ++i) w += __float_as_uint(fminf(fmaf(y[i], r, FINE) + (WHOLE - FINE), WHOLE + 7.f)) << (4 * i);
    return w;
}

// A turned key as the sum of two float32, the first the nearest to the sum (what a float32 rounding would drop decides which code a number
// next to a border between two gets, and which scale): products with their errors by fused multiply-add, the sum with its error as Knuth's
// (The Art of Computer Programming 2, 4.2.2). Each operation is named, so that the compiler cannot fuse a product into the sum whose error is
// taken behind it. What is left out is the roundings of the errors' sum, some 2^-46 of the pair's size. x the channel's own number, o its partner's.
__device__ __forceinline__ void kv4_turn2(float& x, float& lo, float o, float2 cs, bool second) {
    o = second ? o : -o;
    const float p = __fmul_rn(x, cs.x), q = __fmul_rn(o, cs.y), h = __fadd_rn(p, q), b = __fsub_rn(h, p);
    const float rest = __fadd_rn(__fsub_rn(p, __fsub_rn(h, b)), __fsub_rn(q, b));
    const float l = __fadd_rn(rest, __fadd_rn(__fmaf_rn(x, cs.x, -p), __fmaf_rn(o, cs.y, -q)));
    x = __fadd_rn(h, l);
    lo = __fsub_rn(l, __fsub_rn(x, h));
}

// The key whose maximum over a group names its m, of such numbers: the first part's magnitude, then how far the second goes beyond it, "not
// negative" in the lowest bit.
__device__ __forceinline__ unsigned long long kv4_most2(float hi, float lo) {
    const unsigned b = __float_as_uint(hi);
    const float beyond = (b >> 31 ? -lo : lo) + 0.f;                   // (no -0)
    const unsigned l = __float_as_uint(beyond), order = l >> 31 ? ~l : l | 0x80000000u;
    return (unsigned long long)(b & 0x7fffffffu) << 32 | (order & ~1u) | (b >> 31 ^ 1u);
}

// The scale from that key. Only where the first part lies half way between two scales does the second decide.
__device__ __forceinline__ float kv4_make_scale2(unsigned long long most) {
    const unsigned size = (unsigned)(most >> 32), order = (unsigned)most & ~1u;
    if (size >= 0x7f800000u) return __uint_as_float(0x7fc00000u);
    if (size < 0x05000000u) return 0.f;
    unsigned d = size - (3u << 23);
    const unsigned even = (d >> 19) & 1u, up = order > 0x80000000u ? 1u : order < 0x80000000u ? 0u : even;
    d = (d + 0x3ffffu + ((d & 0x7ffffu) == 0x40000u ? up : even)) & 0xfff80000u;
    return __uint_as_float(d | (unsigned)(most & 1u) << 31);
}

// Codes of such numbers, hi + lo. s is the whole number nearest to hi / d by the hardware's reciprocal; what it leaves, hi - s d (exact) and
// lo, is then compared with half a step.
template <int N>
__device__ __noinline__ unsigned kv4_codes2(const float (&hi)[N], const float (&lo)[N], float d) {
    if (!(fabsf(d) > 0.f)) return 0x88888888u;
    constexpr float WHOLE = 12582912.f;
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(d));
    const float half = 0.5f * fabsf(d), toward = d < 0.f ? -1.f : 1.f;
    unsigned w = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const float t = fmaf(hi[i], r, WHOLE);
        float s = t - WHOLE;
        const float left = fmaf(-s, d, hi[i]);
        const float over = (fabsf(left) - half) + (left < 0.f ? -lo[i] : lo[i]);
        if (over > 0.f || (over == 0.f && (__float_as_uint(t) & 1u))) s += left < 0.f ? -toward : toward;
        w |= (__float_as_uint(fminf(fmaxf(s, -8.f), 7.f) + (WHOLE + 8.f)) & 15u) << (4 * i);
    }
    return w;
}

// channel c of a head, turned: `x` the channel's own number, `o` its partner's, c and s of the pair's angle
__device__ __forceinline__ float kv4_turn(float x, float o, float2 cs, bool second) { return second ? fmaf(x, cs.x, o * cs.y) : fmaf(x, cs.x, -o * cs.y); }

// Scale and codes of this thread's eight channels of a key (from c0 on, those below rot turned), exactly; the four lanes of a group, `mask`, together.
template <typename T>
__device__ __noinline__ void kv4_key_again(const T* p, const float2* turn, int c0, int rot, int half, unsigned mask, float& d, unsigned& codes) {
    float y[8], lo[8];
    unsigned long long m = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const int c = c0 + j;
        y[j] = gb_to_float(p[c]);
        lo[j] = 0.f;
        if (c < rot) kv4_turn2(y[j], lo[j], gb_to_float(p[c >= half ? c - half : c + half]), turn[c >= half ? c - half : c], c >= half);
        m = max(m, kv4_most2(y[j], lo[j]));
    }
    m = max(m, __shfl_xor_sync(mask, m, 1));
    m = max(m, __shfl_xor_sync(mask, m, 2));
    d = kv4_make_scale2(m);
    codes = kv4_codes2(y, lo, d);
}

// The page of a slot; shift: of a page size that is a power of two, else -1.
__device__ __forceinline__ int kv4_page(int slot, int page_size, int shift) { return shift >= 0 ? slot >> shift : slot / page_size; }
static int kv4_page_shift(int page_size) {
    int shift = 0;
    while (shift < 30 && (1 << shift) < page_size) ++shift;
    return (1 << shift) == page_size ? shift : -1;
}

struct Kv4WriteArgs {
    const void* qkv;
    long long qkv_stride;
    void* q;
    long long q_stride;
    const float2* table;
    const int* positions;
    const int* slots;
    unsigned char* kcache;
    unsigned char* vcache;
    int nh, nkv, hd, rot, max_pos, page_size, page_shift, write_kv;
    long long num_slots;
    int* status;
    int units_v, units_k, units_q;           // work items of a row: values, keys, queries
    Kv4Div by_w, by_g, by_pairs;             // pairs of groups, groups, items of a query head
};

// One row a block (blockIdx.y: its items KV4_THREADS at a time). Work items, one a thread: values (four channels in each of two neighbouring
// groups: a word of codes), eight lanes to a pair of groups; keys (eight channels of a group: a word), four lanes to a group; queries
// (eight pairs of channels, or twice eight channels that do not turn). WIDE: everything starts on 16 bytes and rot / 2 is a multiple of 8.
template <typename T, bool WIDE>
__global__ void __launch_bounds__(KV4_THREADS) kv4_write_kernel(const Kv4WriteArgs a) {
    gb_pdl_launch_dependents();
    gb_pdl_wait();
    const int row = blockIdx.x, item = blockIdx.y * KV4_THREADS + threadIdx.x;
    if (item >= a.units_v + a.units_k + a.units_q) return;
    // (asked for first and looked at behind the row's own loads, which do not depend on them)
    const int pos = a.positions[row], slot = a.write_kv ? a.slots[row] : 0;
    const int hd = a.hd, G = hd / KV4_GROUP, half = a.rot / 2, lane = threadIdx.x & 31;
    const T* base = (const T*)a.qkv + (size_t)row * a.qkv_stride;
    auto turns = [&]() { return a.table != nullptr && pos < a.max_pos; };
    auto stores = [&]() { return slot >= 0 && slot < a.num_slots; };
    auto report = [&]() {
        if (item == 0 && pos >= 0) {
            const int bad = (a.table != nullptr && !turns() ? GB_STATUS_BAD_POSITION : 0) | (a.write_kv && !stores() ? GB_STATUS_BAD_SLOT : 0);
            if (bad) atomicOr(a.status, bad);
        }
    };

    if (item < a.units_v) {
        const int u = item & 7, h = a.by_w.of(item >> 3), w = (item >> 3) - h * (int)a.by_w.d;
        const bool two = 2 * w + 1 < G;
        const T* p = base + (size_t)(a.nh + a.nkv + h) * hd + 64 * w + 4 * u;
        float y0[4], y1[4] = {0.f, 0.f, 0.f, 0.f};
        kv4_load<T, 4, WIDE>(p, y0);
        if (two) kv4_load<T, 4, WIDE>(p + 32, y1);
        report();
        if (pos < 0 || !stores()) return;    // a padding row, or a bad slot (the same for all items of a row: no lane of a group is missing)
        const int page = kv4_page(slot, a.page_size, a.page_shift), off = slot - page * a.page_size, r = off % KV4_TILE;
        float high0, low0, high1, low1;
        kv4_ends(y0, high0, low0);
        kv4_ends(y1, high1, low1);
        const unsigned mask = 0xffu << (lane & 24);
#pragma unroll
        for (int o = 1; o < 8; o <<= 1) {
            high0 = kv4_max_nan(high0, __shfl_xor_sync(mask, high0, o));
            low0 = kv4_min_nan(low0, __shfl_xor_sync(mask, low0, o));
            high1 = kv4_max_nan(high1, __shfl_xor_sync(mask, high1, o));
            low1 = kv4_min_nan(low1, __shfl_xor_sync(mask, low1, o));
        }
        const float d0 = kv4_make_scale(high0, low0), d1 = kv4_make_scale(high1, low1);
        unsigned char* tile = a.vcache + kv4_tile(page, h, off, a.nkv, a.page_size) * kv4_tile_bytes(hd);
        unsigned char* codes = tile + r * (hd / 2) + (u * G + 2 * w) * 2;
        unsigned short* scales = reinterpret_cast<unsigned short*>(tile + 8 * hd) + r * G + 2 * w;
        unsigned c0, c1;
        if (sizeof(T) == 2) {
            c0 = kv4_codes_bf16(y0, d0);
            c1 = kv4_codes_bf16(y1, d1);
        } else {                             // (the quotient of a float32 may have been rounded to half way)
            const float none[4] = {0.f, 0.f, 0.f, 0.f};
            float near;
            c0 = kv4_codes(y0, d0, near);
            if (near == 0.5f) c0 = kv4_codes2(y0, none, d0);
            c1 = kv4_codes(y1, d1, near);
            if (near == 0.5f) c1 = kv4_codes2(y1, none, d1);
        }
        c0 &= 0xffffu;
        c1 &= 0xffffu;
        if (two && G % 2 == 0) {
            *reinterpret_cast<unsigned*>(codes) = c0 | c1 << 16;
            if (u == 0) *reinterpret_cast<unsigned*>(scales) = __float_as_uint(d0) >> 16 | (__float_as_uint(d1) & 0xffff0000u);
        } else {
            *reinterpret_cast<unsigned short*>(codes) = (unsigned short)c0;
            if (u == 0) scales[0] = (unsigned short)(__float_as_uint(d0) >> 16);
            if (two) {
                *reinterpret_cast<unsigned short*>(codes + 2) = (unsigned short)c1;
                if (u == 0) scales[1] = (unsigned short)(__float_as_uint(d1) >> 16);
            }
        }
        return;
    }
    if (item < a.units_v + a.units_k) {
        const int k = item - a.units_v, t = k & 3, h = a.by_g.of(k >> 2), g = (k >> 2) - h * G, c0 = KV4_GROUP * g + 8 * t;
        const T* p = base + (size_t)(a.nh + h) * hd;
        const bool second = c0 >= half;
        const int first = second ? c0 - half : c0;      // (WIDE: of the pairs that these channels belong to)
        float y[8], o[8];
        kv4_load<T, 8, WIDE>(p + c0, y);
        if (WIDE && a.table != nullptr && c0 < a.rot) kv4_load<T, 8, WIDE>(p + (second ? first : first + half), o);
        if (pos < 0 || !stores()) return;
        const int page = kv4_page(slot, a.page_size, a.page_shift), off = slot - page * a.page_size, r = off % KV4_TILE;
        const unsigned mask = 0xfu << (lane & 28);
        const bool turn_them = turns() && c0 < a.rot;
        const float2* turn = a.table + (size_t)pos * half;
        float off_by = turn_them ? 1e-37f : 0.f;         // what a bound on the turned keys' roundings goes by
        if (turn_them) {
            if (WIDE) {
                const float4* cs = reinterpret_cast<const float4*>(turn + first);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float4 f = cs[j];
                    const float s0 = second ? f.y : -f.y, s1 = second ? f.w : -f.w;
                    const float q0 = o[2 * j] * s0, q1 = o[2 * j + 1] * s1;
                    off_by = fmaxf(off_by, fmaxf(fabsf(q0), fabsf(q1)));
                    y[2 * j] = fmaf(y[2 * j], f.x, q0);
                    y[2 * j + 1] = fmaf(y[2 * j + 1], f.z, q1);
                }
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const int c = c0 + j;
                    if (c >= a.rot) continue;
                    const bool late = c >= half;
                    const float2 cs = turn[late ? c - half : c];
                    const float q = gb_to_float(p[late ? c - half : c + half]) * (late ? cs.y : -cs.y);
                    off_by = fmaxf(off_by, fabsf(q));
                    y[j] = fmaf(y[j], cs.x, q);
                }
            }
        }
        float high, low, near;
        kv4_ends(y, high, low);
#pragma unroll
        for (int x = 1; x < 4; x <<= 1) {
            high = kv4_max_nan(high, __shfl_xor_sync(mask, high, x));
            low = kv4_min_nan(low, __shfl_xor_sync(mask, low, x));
            off_by = fmaxf(off_by, __shfl_xor_sync(mask, off_by, x));
        }
        float d = kv4_make_scale(high, low);
        unsigned codes = kv4_codes(y, d, near);
        // Where what the roundings come to could change the sign or the size of the scale, or a code, the group is held once more, exactly.
        const float size = fmaxf(high, -low), bound = 0x1p-22f * fmaxf(off_by, size);
        const bool unsure = off_by > 0.f ? fabsf(high + low) <= 2.f * bound || kv4_five(__float_as_uint(size - bound)) != kv4_five(__float_as_uint(size + bound)) ||
                                               (0.5f - near) * fabsf(d) <= 2.f * bound
                                         : sizeof(T) == 4 && near == 0.5f;
        if (__ballot_sync(mask, unsure)) kv4_key_again<T>(p, turn, c0, turn_them ? a.rot : 0, half, mask, d, codes);
        unsigned char* tile = a.kcache + kv4_tile(page, h, off, a.nkv, a.page_size) * kv4_tile_bytes(hd);
        *reinterpret_cast<unsigned*>(tile + r * (hd / 2) + (t * G + g) * 4) = codes;
        if (t == 0) reinterpret_cast<unsigned short*>(tile + 8 * hd)[r * G + g] = (unsigned short)(__float_as_uint(d) >> 16);
        return;
    }

    // queries: of a head, or (WIDE, an even number of them) of two heads nh / 2 apart, which turn by the same angles
    const int k = item - a.units_v - a.units_k, h = a.by_pairs.of(k), i = k - h * (int)a.by_pairs.d;
    const T* p = base + (size_t)h * hd;
    T* to = (T*)a.q + (size_t)row * a.q_stride + (size_t)h * hd;
    if (WIDE) {
        const bool twins = a.nh % 2 == 0;
        const size_t twin = (size_t)(a.nh / 2) * hd;
        if (8 * i < half) {
            Kv4Asked<T, 8> x[4];
            x[0].ask(p + 8 * i);
            x[1].ask(p + 8 * i + half);
            if (twins) {
                x[2].ask(p + twin + 8 * i);
                x[3].ask(p + twin + 8 * i + half);
            }
            report();
            if (pos < 0) return;
            const float4* cs = reinterpret_cast<const float4*>(a.table + (size_t)pos * half + 8 * i);
            float4 angle[4];
            const bool turn = turns();
            if (turn) {
#pragma unroll
                for (int j = 0; j < 4; ++j) angle[j] = cs[j];
            }
#pragma unroll
            for (int y = 0; y < 2; ++y) {
                if (y == 1 && !twins) break;
                float x0[8], x1[8];
                x[2 * y].get(x0);
                x[2 * y + 1].get(x1);
                if (turn) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const float2 c = j % 2 ? make_float2(angle[j / 2].z, angle[j / 2].w) : make_float2(angle[j / 2].x, angle[j / 2].y);
                        const float z0 = kv4_turn(x0[j], x1[j], c, false), z1 = kv4_turn(x1[j], x0[j], c, true);
                        x0[j] = z0;
                        x1[j] = z1;
                    }
                }
                kv4_store<T, 8, WIDE>(to + y * twin + 8 * i, x0);
                kv4_store<T, 8, WIDE>(to + y * twin + 8 * i + half, x1);
            }
        } else {
            const int c = a.rot + 8 * (i - half / 8), second = (hd - a.rot) / 2;
            constexpr int EACH = (int)sizeof(T) / 2;
            uint4 raw[4 * EACH];
            auto at = [&](int j) { return c + (size_t)(j / EACH % 2) * second + (size_t)(j / EACH / 2) * twin; };
#pragma unroll
            for (int j = 0; j < 4 * EACH; ++j)
                if (j < 2 * EACH || twins) raw[j] = reinterpret_cast<const uint4*>(p + at(j))[j % EACH];
            report();
            if (pos < 0) return;
#pragma unroll
            for (int j = 0; j < 4 * EACH; ++j)
                if (j < 2 * EACH || twins) reinterpret_cast<uint4*>(to + at(j))[j % EACH] = raw[j];
        }
        return;
    }
    report();
    if (pos < 0) return;
    if (i < half) {                          // one pair, or one channel, a thread
        const float x0 = gb_to_float(p[i]), x1 = gb_to_float(p[i + half]);
        const bool turn = turns();
        const float2 cs = turn ? a.table[(size_t)pos * half + i] : make_float2(1.f, 0.f);
        to[i] = gb_from_float<T>(turn ? kv4_turn(x0, x1, cs, false) : x0);
        to[i + half] = gb_from_float<T>(turn ? kv4_turn(x1, x0, cs, true) : x1);
    } else {
        const int c = a.rot + i - half;
        to[c] = p[c];
    }
}

// qkv [n, (nh + 2 nkv) hd] (rows qkv_stride numbers apart) -> q [n, nh hd] (rows q_stride apart; may be the query columns of qkv itself),
// and the cache at each row's slot. Rows of position < 0 are padding and touch nothing; a bad slot or position is reported and the
// store or the rotation left out.
GB_EXPORT int gb_kv4_write(const void* qkv, long long qkv_stride, int dtype, void* q, long long q_stride, const float* cos_sin,
                           const int* positions, const int* slots, void* kcache, void* vcache, int n, int nh, int nkv, int hd, int rot,
                           int max_pos, int page_size, long long num_pages, int write_kv, int* status, cudaStream_t stream) {
    KV4_REQUIRE_SIZES("gb_kv4_write")
    GB_REQUIRE(n >= 0 && nh > 0 && rot >= 0 && rot <= hd && rot % 2 == 0, "gb_kv4_write: bad sizes (rows %d, heads %d, rotary size %d of %d)", n, nh, rot, hd);
    GB_REQUIRE(dtype == GB_F32 || dtype == GB_BF16, "gb_kv4_write: unsupported dtype %d", dtype);
    GB_REQUIRE(((uintptr_t)kcache | (uintptr_t)vcache) % 16 == 0, "gb_kv4_write: the cache must be 16-byte aligned");
    GB_REQUIRE(rot == 0 || cos_sin != nullptr, "gb_kv4_write: a rotation needs its table");
    if (n == 0) return 0;
    const int size = dtype == GB_F32 ? 4 : 2, G = hd / KV4_GROUP;
    const bool wide = rot % 16 == 0 && ((uintptr_t)qkv | (uintptr_t)q | (rot ? (uintptr_t)cos_sin : 0)) % 16 == 0 && (qkv_stride * size) % 16 == 0 &&
                      (q_stride * size) % 16 == 0;
    Kv4WriteArgs a = {};
    a.qkv = qkv; a.qkv_stride = qkv_stride; a.q = q; a.q_stride = q_stride; a.table = rot ? (const float2*)cos_sin : nullptr;
    a.positions = positions; a.slots = slots; a.kcache = (unsigned char*)kcache; a.vcache = (unsigned char*)vcache; a.nh = nh;
    a.nkv = nkv; a.hd = hd; a.rot = rot; a.max_pos = max_pos; a.page_size = page_size; a.page_shift = kv4_page_shift(page_size); a.write_kv = write_kv;
    a.num_slots = num_pages * page_size; a.status = status;
    a.units_v = write_kv ? nkv * ((G + 1) / 2) * 8 : 0;
    a.units_k = write_kv ? nkv * G * 4 : 0;
    // (channels that do not turn are copied only where the queries go somewhere else)
    const bool in_place = q == qkv && q_stride == qkv_stride;
    const int pairs = wide ? rot / 16 + (in_place ? 0 : (hd - rot) / 16) : rot / 2 + (in_place ? 0 : hd - rot);
    a.units_q = (wide && nh % 2 == 0 ? nh / 2 : nh) * pairs;
    a.by_w = Kv4Div((G + 1) / 2);
    a.by_g = Kv4Div(G);
    a.by_pairs = Kv4Div(pairs > 0 ? pairs : 1);
    const int units = a.units_v + a.units_k + a.units_q;
    if (units == 0) return 0;
    const dim3 grid(n, gb_ceil_div(units, KV4_THREADS)), block(KV4_THREADS);
    if (dtype == GB_F32)
        gb_launch(GB_PDL_ELEMENTWISE, wide ? kv4_write_kernel<float, true> : kv4_write_kernel<float, false>, grid, block, 0, stream, a);
    else
        gb_launch(GB_PDL_ELEMENTWISE, wide ? kv4_write_kernel<__nv_bfloat16, true> : kv4_write_kernel<__nv_bfloat16, false>, grid, block, 0, stream, a);
    return gb_check_launch("gb_kv4_write");
}

// Eight neighbouring channels (part t of four of group g) of a key, or of a value: their codes as a word, the lowest channel's first.
__device__ __forceinline__ unsigned kv4_word(const unsigned char* tile, int hd, int r, int g, int t, bool value) {
    const int G = hd / KV4_GROUP;
    const unsigned char* row = tile + r * (hd / 2);
    if (!value) return *reinterpret_cast<const unsigned*>(row + (t * G + g) * 4);
    return *reinterpret_cast<const unsigned short*>(row + (2 * t * G + g) * 2) | (unsigned)*reinterpret_cast<const unsigned short*>(row + ((2 * t + 1) * G + g) * 2) << 16;
}

// What such a word stands for, as eight bfloat16 (two a word): codes under 0x4300 are 128 + s + 8, and the product with the scale is exact.
__device__ __forceinline__ void kv4_eight(unsigned w, unsigned short scale, uint32_t (&x)[4]) {
    const unsigned d2 = scale | (unsigned)scale << 16, c2 = 0x43084308u;
    uint32_t y[4];                           // channels i and i + 4
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const unsigned u = (w >> (4 * i) & 0x000f000fu) | 0x43004300u;
        const __nv_bfloat162 v = __hmul2(__hsub2(*reinterpret_cast<const __nv_bfloat162*>(&u), *reinterpret_cast<const __nv_bfloat162*>(&c2)),
                                         *reinterpret_cast<const __nv_bfloat162*>(&d2));
        y[i] = *reinterpret_cast<const uint32_t*>(&v);
    }
    x[0] = __byte_perm(y[0], y[1], 0x5410);
    x[1] = __byte_perm(y[2], y[3], 0x5410);
    x[2] = __byte_perm(y[0], y[1], 0x7632);
    x[3] = __byte_perm(y[2], y[3], 0x7632);
}
__device__ __forceinline__ void kv4_put(__nv_bfloat16* p, const uint32_t (&x)[4]) { *reinterpret_cast<uint4*>(p) = make_uint4(x[0], x[1], x[2], x[3]); }
__device__ __forceinline__ void kv4_put(float* p, const uint32_t (&x)[4]) {
#pragma unroll
    for (int i = 0; i < 4; i += 2)
        *reinterpret_cast<uint4*>(p + 2 * i) = make_uint4(x[i] << 16, x[i] & 0xffff0000u, x[i + 1] << 16, x[i + 1] & 0xffff0000u);
}

// One row a block (blockIdx.y: its items KV4_THREADS at a time), eight neighbouring channels of a key and of its value a thread.
template <typename T>
__global__ void __launch_bounds__(KV4_THREADS) kv4_read_kernel(const unsigned char* __restrict__ kcache, const unsigned char* __restrict__ vcache,
                                                              const int* __restrict__ slots, T* __restrict__ k, T* __restrict__ v, int nkv,
                                                              int hd, int page_size, int page_shift, long long num_slots, Kv4Div by_g, int* __restrict__ status) {
    gb_pdl_launch_dependents();
    gb_pdl_wait();
    const int row = blockIdx.x, slot = slots[row], item = blockIdx.y * KV4_THREADS + threadIdx.x;
    if (slot < 0 || item >= nkv * (hd / 8)) return;
    if (slot >= num_slots) {
        if (item == 0) atomicOr(status, GB_STATUS_BAD_SLOT);
        return;
    }
    const int G = hd / KV4_GROUP, t = item & 3, h = by_g.of(item >> 2), g = (item >> 2) - h * G;
    const int page = kv4_page(slot, page_size, page_shift), off = slot - page * page_size, r = off % KV4_TILE;
    const long long at = kv4_tile(page, h, off, nkv, page_size) * kv4_tile_bytes(hd);
    const unsigned key = kv4_word(kcache + at, hd, r, g, t, false), value = kv4_word(vcache + at, hd, r, g, t, true);
    const int scale = 8 * hd + (r * G + g) * 2;
    const unsigned short dk = *reinterpret_cast<const unsigned short*>(kcache + at + scale), dv = *reinterpret_cast<const unsigned short*>(vcache + at + scale);
    const size_t to = ((size_t)row * nkv + h) * hd + KV4_GROUP * g + 8 * t;
    uint32_t x[4];
    kv4_eight(key, dk, x);
    kv4_put(k + to, x);
    kv4_eight(value, dv, x);
    kv4_put(v + to, x);
}

GB_EXPORT int gb_kv4_read(const void* kcache, const void* vcache, const int* slots, void* k, void* v, int dtype, int n, int nkv, int hd,
                          int page_size, long long num_pages, int* status, cudaStream_t stream) {
    KV4_REQUIRE_SIZES("gb_kv4_read")
    GB_REQUIRE(dtype == GB_F32 || dtype == GB_BF16, "gb_kv4_read: unsupported dtype %d", dtype);
    GB_REQUIRE(((uintptr_t)kcache | (uintptr_t)vcache | (uintptr_t)k | (uintptr_t)v) % 16 == 0, "gb_kv4_read: tensors must be 16-byte aligned");
    if (n <= 0) return 0;
    const dim3 grid(n, gb_ceil_div(nkv * (hd / 8), KV4_THREADS)), block(KV4_THREADS);
    const unsigned char *kc = (const unsigned char*)kcache, *vc = (const unsigned char*)vcache;
    const Kv4Div by_g(hd / KV4_GROUP);
    if (dtype == GB_F32)
        gb_launch(GB_PDL_ELEMENTWISE, kv4_read_kernel<float>, grid, block, 0, stream, kc, vc, slots, (float*)k, (float*)v, nkv, hd, page_size,
                  kv4_page_shift(page_size), num_pages * page_size, by_g, status);
    else
        gb_launch(GB_PDL_ELEMENTWISE, kv4_read_kernel<__nv_bfloat16>, grid, block, 0, stream, kc, vc, slots, (__nv_bfloat16*)k, (__nv_bfloat16*)v, nkv,
                  hd, page_size, kv4_page_shift(page_size), num_pages * page_size, by_g, status);
    return gb_check_launch("gb_kv4_read");
}

// Pages of 4 bits that the rows of a step see, as numbers into pages of the same ids: one block a page of a request and kv head.
// Numbers of tokens outside the request's range (before its first row's window, behind its last row) that are NaN become zero: the
// kernels that read the pages multiply what they mask by zero. (Of two requests that share a page, a NaN in which lies before the window of one and
// in sight of the other, either may have its way.) Bound by the latency of a page's few loads: 7 us for 4,096 tokens of 8 heads of 128, 21 MB, 17 of them written.
template <typename T>
__global__ void __launch_bounds__(KV4_THREADS) kv4_expand_kernel(const unsigned char* __restrict__ kcache, const unsigned char* __restrict__ vcache,
                                                                T* __restrict__ k, T* __restrict__ v, const int* __restrict__ block_tables, int max_pages,
                                                                const int* __restrict__ seq_first_row, const int* __restrict__ seq_start_pos, int nkv,
                                                                int hd, int page_size, long long num_pages, int window, Kv4Div by_row,
                                                                int* __restrict__ status) {
    gb_pdl_launch_dependents();
    gb_pdl_wait();
    const int seq = blockIdx.z, start = seq_start_pos[seq], rows = seq_first_row[seq + 1] - seq_first_row[seq], h = blockIdx.y;
    if (start < 0 || rows <= 0) return;
    const long long end = (long long)start + rows, first = gb_first_key(start, window > 0 ? window : 0);
    const long long begin = (long long)blockIdx.x * page_size;
    if (end > (long long)gridDim.x * page_size && threadIdx.x == 0 && h == 0 && blockIdx.x == 0) atomicOr(status, GB_STATUS_BAD_POSITION);      // tokens that no block unpacks
    if (begin >= end || begin + page_size <= first) return;
    const long long page = block_tables[(size_t)seq * max_pages + blockIdx.x];
    if (page < 0 || page >= num_pages) {
        if (threadIdx.x == 0 && h == 0) atomicOr(status, GB_STATUS_BAD_SLOT);
        return;
    }
    const int G = hd / KV4_GROUP, per_row = hd / 8;                 // items of a token
    const long long head = page * nkv + h;
    const bool inside = begin >= first && begin + page_size <= end;
    const unsigned char* const keys = kcache + head * (page_size / KV4_TILE) * kv4_tile_bytes(hd);
    const unsigned char* const values = vcache + head * (page_size / KV4_TILE) * kv4_tile_bytes(hd);
#pragma unroll 2
    for (int i = threadIdx.x; i < page_size * per_row; i += KV4_THREADS) {      // eight channels of a key and of its value
        const int off = by_row.of(i), c = i - off * per_row, t = c & 3, g = c >> 2, r = off % KV4_TILE;
        const int tile = off / KV4_TILE * kv4_tile_bytes(hd), scale = tile + 8 * hd + (r * G + g) * 2;
        const unsigned key = kv4_word(keys + tile, hd, r, g, t, false), value = kv4_word(values + tile, hd, r, g, t, true);
        unsigned short dk = *reinterpret_cast<const unsigned short*>(keys + scale), dv = *reinterpret_cast<const unsigned short*>(values + scale);
        if (!inside && (begin + off < first || begin + off >= end)) {
            if ((dk & 0x7fffu) > 0x7f80u) dk = 0;
            if ((dv & 0x7fffu) > 0x7f80u) dv = 0;
        }
        const size_t to = (size_t)(head * page_size + off) * hd + 8 * c;
        uint32_t x[4];
        kv4_eight(key, dk, x);
        kv4_put(k + to, x);
        kv4_eight(value, dv, x);
        kv4_put(v + to, x);
    }
}

GB_EXPORT int gb_kv4_expand(const void* kcache, const void* vcache, void* k, void* v, int dtype, const int* block_tables, int max_pages,
                            const int* seq_first_row, const int* seq_start_pos, int num_seqs, int reach_pages, int nkv, int hd, int page_size,
                            long long num_pages, int window, int* status, cudaStream_t stream) {
    KV4_REQUIRE_SIZES("gb_kv4_expand")
    GB_REQUIRE(dtype == GB_F32 || dtype == GB_BF16, "gb_kv4_expand: unsupported dtype %d", dtype);
    GB_REQUIRE(((uintptr_t)kcache | (uintptr_t)vcache | (uintptr_t)k | (uintptr_t)v) % 16 == 0, "gb_kv4_expand: tensors must be 16-byte aligned");
    GB_REQUIRE(num_seqs >= 0 && num_seqs <= 65535 && nkv <= 65535 && max_pages > 0, "gb_kv4_expand: bad batch shape");
    const int pages = reach_pages < max_pages ? reach_pages : max_pages;
    if (num_seqs == 0 || pages <= 0) return 0;
    const dim3 grid(pages, nkv, num_seqs), block(KV4_THREADS);
    const Kv4Div by_row(hd / 8);
    const unsigned char *kc = (const unsigned char*)kcache, *vc = (const unsigned char*)vcache;
    if (dtype == GB_F32)
        gb_launch(GB_PDL_ELEMENTWISE, kv4_expand_kernel<float>, grid, block, 0, stream, kc, vc, (float*)k, (float*)v, block_tables, max_pages,
                  seq_first_row, seq_start_pos, nkv, hd, page_size, num_pages, window, by_row, status);
    else
        gb_launch(GB_PDL_ELEMENTWISE, kv4_expand_kernel<__nv_bfloat16>, grid, block, 0, stream, kc, vc, (__nv_bfloat16*)k, (__nv_bfloat16*)v,
                  block_tables, max_pages, seq_first_row, seq_start_pos, nkv, hd, page_size, num_pages, window, by_row, status);
    return gb_check_launch("gb_kv4_expand");
}
