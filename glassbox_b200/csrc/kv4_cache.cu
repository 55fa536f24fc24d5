// Writing a cache in 4 bits and reading it back (layout: kv4.cuh). Three kernels:
//   kv4_write   rotates the queries and keys of a step's rows, rounds keys and values to 4 bits and stores them in their pages;
//   kv4_read    what the cache holds for given slots, as numbers;
//   kv4_expand  the pages that a step's requests see, as pages of bfloat16 or float32 that the prompt kernels read.
// All three only move memory. The sums that matter are bytes: a row of a wide layout (32/8 heads of 128, bfloat16) brings 12 KB in, 8 KB
// of queries out and 1.1 KB of cache out.
//
// The rounding, for numbers y of a group (float32, after the rotation): one 32-bit key per number, its magnitude's bits with "not
// negative" in the lowest, has the group's m as its maximum, infinities and NaN above every number; m's bits less 3 in the
// exponent, rounded to four bits after the leading one, are |d|. The quotient y / d is the product with the reciprocal and one
// correction by the remainder (exact in a fused multiply-add), so that a number half way between two codes is told as such: with bfloat16
// values that is one in dozens, and ties go to the even code.
#include "kv4.cuh"

#include <type_traits>

constexpr int KV4_THREADS = 256;

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

// The key whose maximum over a group names its m (see above), over N numbers of this thread.
template <int N>
__device__ __forceinline__ unsigned kv4_most(const float (&y)[N]) {
    unsigned most = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const unsigned b = __float_as_uint(y[i]);
        most = max(most, (b << 1) | (b >> 31 ^ 1u));
    }
    return most;
}

// The scale of a group from that key, as float32: zero, NaN, or a number of five significant bits.
__device__ __forceinline__ float kv4_make_scale(unsigned most) {
    const unsigned size = most >> 1;
    if (size >= 0x7f800000u) return __uint_as_float(0x7fc00000u);
    if (size < 0x05000000u) return 0.f;                                    // 2^-117
    unsigned d = size - (3u << 23);
    d = (d + 0x3ffffu + ((d >> 19) & 1u)) & 0xfff80000u;                   // four bits after the leading one, ties to even
    return __uint_as_float(d | (most & 1u) << 31);                         // (m positive: d negative)
}

// Codes s + 8 of N numbers, N nibbles from the low end on.
template <int N>
__device__ __forceinline__ unsigned kv4_codes(const float (&y)[N], float d) {
    if (!(fabsf(d) > 0.f)) return 0x88888888u;                             // nothing, or NaN: s = 0
    const float r = 1.0f / d;
    unsigned w = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        float q = y[i] * r;
        q = fmaf(fmaf(-q, d, y[i]), r, q);
        const int s = __float2int_rn(fminf(fmaxf(q, -8.f), 7.f)) + 8;
        w |= (unsigned)s << (4 * i);
    }
    return w;
}

// channel c of a head, turned: `x` the channel's own number, `o` its partner's, c and s of the pair's angle
__device__ __forceinline__ float kv4_turn(float x, float o, float2 cs, bool second) { return second ? fmaf(x, cs.x, o * cs.y) : fmaf(x, cs.x, -o * cs.y); }

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
    int n, nh, nkv, hd, rot, max_pos, page_size, write_kv;
    long long num_slots;
    int* status;
    int units, units_v, units_k, pairs;      // work items of a row: values, keys, then queries; items of a query head
};

// Work items of a row, one a thread: values (four channels in each of two neighbouring groups: a word of codes), eight lanes to a
// pair of groups; keys (eight channels of a group: a word), four lanes to a group; queries (eight pairs of channels, or eight channels
// that do not turn). WIDE: everything starts on 16 bytes and rot / 2 is a multiple of 8.
template <typename T, bool WIDE>
__global__ void __launch_bounds__(KV4_THREADS) kv4_write_kernel(const Kv4WriteArgs a) {
    gb_pdl_launch_dependents();
    gb_pdl_wait();
    const unsigned at = blockIdx.x * KV4_THREADS + threadIdx.x;
    const int row = (int)(at / (unsigned)a.units), item = (int)(at % (unsigned)a.units);
    if (row >= a.n) return;
    const int pos = a.positions[row];
    if (pos < 0) return;                     // a padding row: nothing to turn, nothing to store
    const long long slot = a.write_kv ? a.slots[row] : 0;
    const bool rotate = a.table != nullptr && pos < a.max_pos, store = a.write_kv && slot >= 0 && slot < a.num_slots;
    if (item == 0 && ((a.table != nullptr && !rotate) || (a.write_kv && !store)))
        atomicOr(a.status, (a.table != nullptr && !rotate ? GB_STATUS_BAD_POSITION : 0) | (a.write_kv && !store ? GB_STATUS_BAD_SLOT : 0));
    const int hd = a.hd, G = hd / KV4_GROUP, half = a.rot / 2, lane = threadIdx.x & 31;
    const T* base = (const T*)a.qkv + (size_t)row * a.qkv_stride;
    const float2* turn = rotate ? a.table + (size_t)pos * half : nullptr;

    if (item < a.units_v + a.units_k) {
        if (!store) return;                  // (the same for all items of a row: no lane of a group is missing)
        const int off = (int)(slot % a.page_size);
        const long long page = slot / a.page_size;
        const int r = off % KV4_TILE;
        if (item < a.units_v) {
            const int W = (G + 1) / 2, u = item & 7, w = (item >> 3) % W, h = (item >> 3) / W;
            const bool two = 2 * w + 1 < G;
            const T* p = base + (size_t)(a.nh + a.nkv + h) * hd + 64 * w + 4 * u;
            float y0[4], y1[4] = {0.f, 0.f, 0.f, 0.f};
            kv4_load<T, 4, WIDE>(p, y0);
            if (two) kv4_load<T, 4, WIDE>(p + 32, y1);
            unsigned m0 = kv4_most(y0), m1 = kv4_most(y1);
            const unsigned mask = 0xffu << (lane & 24);
#pragma unroll
            for (int o = 1; o < 8; o <<= 1) {
                m0 = max(m0, __shfl_xor_sync(mask, m0, o));
                m1 = max(m1, __shfl_xor_sync(mask, m1, o));
            }
            const float d0 = kv4_make_scale(m0), d1 = kv4_make_scale(m1);
            unsigned char* tile = a.vcache + kv4_tile(page, h, off, a.nkv, a.page_size) * kv4_tile_bytes(hd);
            unsigned char* codes = tile + r * (hd / 2) + (u * G + 2 * w) * 2;
            unsigned short* scales = reinterpret_cast<unsigned short*>(tile + 8 * hd) + r * G + 2 * w;
            const unsigned c0 = kv4_codes(y0, d0) & 0xffffu, c1 = kv4_codes(y1, d1) & 0xffffu;
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
        const int k = item - a.units_v, t = k & 3, g = (k >> 2) % G, h = (k >> 2) / G, c0 = KV4_GROUP * g + 8 * t;
        const T* p = base + (size_t)(a.nh + h) * hd;
        float y[8];
        kv4_load<T, 8, WIDE>(p + c0, y);
        if (rotate && c0 < a.rot) {
            float o[8];
            if (WIDE) {
                const bool second = c0 >= half;
                const int i = second ? c0 - half : c0;
                kv4_load<T, 8, WIDE>(p + (second ? i : i + half), o);
                const float4* cs = reinterpret_cast<const float4*>(turn + i);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float4 f = cs[j];
                    y[2 * j] = kv4_turn(y[2 * j], o[2 * j], make_float2(f.x, f.y), second);
                    y[2 * j + 1] = kv4_turn(y[2 * j + 1], o[2 * j + 1], make_float2(f.z, f.w), second);
                }
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const int c = c0 + j;
                    if (c >= a.rot) continue;
                    const bool second = c >= half;
                    y[j] = kv4_turn(y[j], gb_to_float(p[second ? c - half : c + half]), turn[second ? c - half : c], second);
                }
            }
        }
        unsigned m = kv4_most(y);
        const unsigned mask = 0xfu << (lane & 28);
        m = max(m, __shfl_xor_sync(mask, m, 1));
        m = max(m, __shfl_xor_sync(mask, m, 2));
        const float d = kv4_make_scale(m);
        unsigned char* tile = a.kcache + kv4_tile(page, h, off, a.nkv, a.page_size) * kv4_tile_bytes(hd);
        *reinterpret_cast<unsigned*>(tile + r * (hd / 2) + (t * G + g) * 4) = kv4_codes(y, d);
        if (t == 0) reinterpret_cast<unsigned short*>(tile + 8 * hd)[r * G + g] = (unsigned short)(__float_as_uint(d) >> 16);
        return;
    }

    // queries
    const int k = item - a.units_v - a.units_k;
    if (k >= a.nh * a.pairs) return;         // (items that fill a row up to a multiple of eight)
    const int h = k / a.pairs, i = k % a.pairs;
    const T* p = base + (size_t)h * hd;
    T* to = (T*)a.q + (size_t)row * a.q_stride + (size_t)h * hd;
    if (WIDE) {
        if (8 * i < half) {
            float x0[8], x1[8], z0[8], z1[8];
            kv4_load<T, 8, WIDE>(p + 8 * i, x0);
            kv4_load<T, 8, WIDE>(p + 8 * i + half, x1);
#pragma unroll
            for (int j = 0; j < 8; ++j) { z0[j] = x0[j]; z1[j] = x1[j]; }
            if (rotate) {
                const float4* cs = reinterpret_cast<const float4*>(turn + 8 * i);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float4 f = cs[j];
                    z0[2 * j] = kv4_turn(x0[2 * j], x1[2 * j], make_float2(f.x, f.y), false);
                    z1[2 * j] = kv4_turn(x1[2 * j], x0[2 * j], make_float2(f.x, f.y), true);
                    z0[2 * j + 1] = kv4_turn(x0[2 * j + 1], x1[2 * j + 1], make_float2(f.z, f.w), false);
                    z1[2 * j + 1] = kv4_turn(x1[2 * j + 1], x0[2 * j + 1], make_float2(f.z, f.w), true);
                }
            }
            kv4_store<T, 8, WIDE>(to + 8 * i, z0);
            kv4_store<T, 8, WIDE>(to + 8 * i + half, z1);
        } else {
            const int c = a.rot + 8 * (i - half / 8);
            float x[8];
            kv4_load<T, 8, WIDE>(p + c, x);
            kv4_store<T, 8, WIDE>(to + c, x);
        }
    } else if (i < half) {                   // one pair, or one channel, a thread
        const float x0 = gb_to_float(p[i]), x1 = gb_to_float(p[i + half]);
        const float2 cs = rotate ? turn[i] : make_float2(1.f, 0.f);
        to[i] = gb_from_float<T>(rotate ? kv4_turn(x0, x1, cs, false) : x0);
        to[i + half] = gb_from_float<T>(rotate ? kv4_turn(x1, x0, cs, true) : x1);
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
    a.positions = positions; a.slots = slots; a.kcache = (unsigned char*)kcache; a.vcache = (unsigned char*)vcache; a.n = n; a.nh = nh;
    a.nkv = nkv; a.hd = hd; a.rot = rot; a.max_pos = max_pos; a.page_size = page_size; a.write_kv = write_kv;
    a.num_slots = num_pages * page_size; a.status = status;
    a.units_v = write_kv ? nkv * ((G + 1) / 2) * 8 : 0;
    a.units_k = write_kv ? nkv * G * 4 : 0;
    // (channels that do not turn are copied only where the queries go somewhere else)
    const bool in_place = q == qkv && q_stride == qkv_stride;
    a.pairs = wide ? rot / 16 + (in_place ? 0 : (hd - rot) / 8) : rot / 2 + (in_place ? 0 : hd - rot);
    a.units = (a.units_v + a.units_k + nh * a.pairs + 7) / 8 * 8;
    if (a.units == 0) return 0;
    GB_REQUIRE((long long)n * a.units < (1ll << 31) - KV4_THREADS, "gb_kv4_write: %d rows are too many for one launch", n);
    const dim3 grid(gb_ceil_div((long long)n * a.units, KV4_THREADS)), block(KV4_THREADS);
    if (dtype == GB_F32)
        gb_launch(GB_PDL_ELEMENTWISE, wide ? kv4_write_kernel<float, true> : kv4_write_kernel<float, false>, grid, block, 0, stream, a);
    else
        gb_launch(GB_PDL_ELEMENTWISE, wide ? kv4_write_kernel<__nv_bfloat16, true> : kv4_write_kernel<__nv_bfloat16, false>, grid, block, 0, stream, a);
    return gb_check_launch("gb_kv4_write");
}

// What eight channels of a key (group g, part t of four) or two times four channels of a value (part u of eight) stand for.
__device__ __forceinline__ void kv4_key8(const unsigned char* tile, int hd, int r, int g, int t, float (&x)[8]) {
    const unsigned w = *reinterpret_cast<const unsigned*>(tile + r * (hd / 2) + (t * (hd / KV4_GROUP) + g) * 4);
    const float d = kv4_scale(tile, hd, r, g);
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = kv4_code(w, j) * d;
}
__device__ __forceinline__ void kv4_value4(const unsigned char* tile, int hd, int r, int g, int u, float (&x)[4]) {
    const unsigned w = *reinterpret_cast<const unsigned short*>(tile + r * (hd / 2) + (u * (hd / KV4_GROUP) + g) * 2);
    const float d = kv4_scale(tile, hd, r, g);
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = kv4_code(w, j) * d;
}

// One thread: eight neighbouring channels of a key or of a value (two of its half words).
template <typename T>
__global__ void __launch_bounds__(KV4_THREADS) kv4_read_kernel(const unsigned char* __restrict__ kcache, const unsigned char* __restrict__ vcache,
                                                              const int* __restrict__ slots, T* __restrict__ k, T* __restrict__ v, int n, int nkv,
                                                              int hd, int page_size, long long num_slots, int* __restrict__ status) {
    gb_pdl_launch_dependents();
    gb_pdl_wait();
    const int per = nkv * (hd / 8);          // items of a row and tensor
    const unsigned at = blockIdx.x * KV4_THREADS + threadIdx.x;
    const int row = (int)(at / (unsigned)(2 * per));
    int item = (int)(at % (unsigned)(2 * per));
    if (row >= n) return;
    const long long slot = slots[row];
    if (slot < 0) return;
    if (slot >= num_slots) {
        if (item == 0) atomicOr(status, GB_STATUS_BAD_SLOT);
        return;
    }
    const bool value = item >= per;
    if (value) item -= per;
    const int G = hd / KV4_GROUP, t = item & 3, g = (item >> 2) % G, h = (item >> 2) / G, off = (int)(slot % page_size), r = off % KV4_TILE;
    const unsigned char* tile = (value ? vcache : kcache) + kv4_tile(slot / page_size, h, off, nkv, page_size) * kv4_tile_bytes(hd);
    float x[8];
    if (value) {
        float lo[4], hi[4];
        kv4_value4(tile, hd, r, g, 2 * t, lo);
        kv4_value4(tile, hd, r, g, 2 * t + 1, hi);
#pragma unroll
        for (int j = 0; j < 4; ++j) { x[j] = lo[j]; x[4 + j] = hi[j]; }
    } else {
        kv4_key8(tile, hd, r, g, t, x);
    }
    Kv4Load<T, 8>::store((value ? v : k) + ((size_t)row * nkv + h) * hd + KV4_GROUP * g + 8 * t, x);
}

GB_EXPORT int gb_kv4_read(const void* kcache, const void* vcache, const int* slots, void* k, void* v, int dtype, int n, int nkv, int hd,
                          int page_size, long long num_pages, int* status, cudaStream_t stream) {
    KV4_REQUIRE_SIZES("gb_kv4_read")
    GB_REQUIRE(dtype == GB_F32 || dtype == GB_BF16, "gb_kv4_read: unsupported dtype %d", dtype);
    GB_REQUIRE(((uintptr_t)kcache | (uintptr_t)vcache | (uintptr_t)k | (uintptr_t)v) % 16 == 0, "gb_kv4_read: tensors must be 16-byte aligned");
    if (n <= 0) return 0;
    const long long items = (long long)n * 2 * nkv * (hd / 8);
    GB_REQUIRE(items < (1ll << 31) - KV4_THREADS, "gb_kv4_read: %d rows are too many for one launch", n);
    const dim3 grid(gb_ceil_div(items, KV4_THREADS)), block(KV4_THREADS);
    const unsigned char *kc = (const unsigned char*)kcache, *vc = (const unsigned char*)vcache;
    if (dtype == GB_F32)
        gb_launch(GB_PDL_ELEMENTWISE, kv4_read_kernel<float>, grid, block, 0, stream, kc, vc, slots, (float*)k, (float*)v, n, nkv, hd, page_size,
                  num_pages * page_size, status);
    else
        gb_launch(GB_PDL_ELEMENTWISE, kv4_read_kernel<__nv_bfloat16>, grid, block, 0, stream, kc, vc, slots, (__nv_bfloat16*)k, (__nv_bfloat16*)v, n,
                  nkv, hd, page_size, num_pages * page_size, status);
    return gb_check_launch("gb_kv4_read");
}

// Pages of 4 bits that the rows of a step see, as numbers into pages of the same ids: one block a page of a request, all heads.
// Numbers of tokens outside the request's range (before its first row's window, behind its last row) that are NaN become zero: the
// kernels that read the pages multiply what they mask by zero.
template <typename T>
__global__ void __launch_bounds__(KV4_THREADS) kv4_expand_kernel(const unsigned char* __restrict__ kcache, const unsigned char* __restrict__ vcache,
                                                                T* __restrict__ k, T* __restrict__ v, const int* __restrict__ block_tables, int max_pages,
                                                                const int* __restrict__ seq_first_row, const int* __restrict__ seq_start_pos, int nkv,
                                                                int hd, int page_size, long long num_pages, int window, int* __restrict__ status) {
    gb_pdl_launch_dependents();
    gb_pdl_wait();
    const int seq = blockIdx.y, start = seq_start_pos[seq], rows = seq_first_row[seq + 1] - seq_first_row[seq];
    if (start < 0 || rows <= 0) return;
    const long long end = (long long)start + rows, first = gb_first_key(start, window > 0 ? window : 0);
    const long long begin = (long long)blockIdx.x * page_size;
    if (begin >= end || begin + page_size <= first) return;
    const long long page = block_tables[(size_t)seq * max_pages + blockIdx.x];
    if (page < 0 || page >= num_pages) {
        if (threadIdx.x == 0) atomicOr(status, GB_STATUS_BAD_SLOT);
        return;
    }
    const int G = hd / KV4_GROUP, per = page_size * G * 4;         // items of a head and tensor
    for (int i = threadIdx.x; i < 2 * nkv * per; i += KV4_THREADS) {
        const bool value = i >= nkv * per;
        int item = value ? i - nkv * per : i;
        const int t = item & 3;
        item >>= 2;
        const int g = item % G;
        item /= G;
        const int off = item % page_size, h = item / page_size, r = off % KV4_TILE;
        const unsigned char* tile = (value ? vcache : kcache) + kv4_tile(page, h, off, nkv, page_size) * kv4_tile_bytes(hd);
        float x[8];
        if (value) {
            float lo[4], hi[4];
            kv4_value4(tile, hd, r, g, 2 * t, lo);
            kv4_value4(tile, hd, r, g, 2 * t + 1, hi);
#pragma unroll
            for (int j = 0; j < 4; ++j) { x[j] = lo[j]; x[4 + j] = hi[j]; }
        } else {
            kv4_key8(tile, hd, r, g, t, x);
        }
        if ((begin + off < first || begin + off >= end) && !(x[0] == x[0])) {
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = 0.f;
        }
        Kv4Load<T, 8>::store((value ? v : k) + (((size_t)page * nkv + h) * page_size + off) * hd + KV4_GROUP * g + 8 * t, x);
    }
}

GB_EXPORT int gb_kv4_expand(const void* kcache, const void* vcache, void* k, void* v, int dtype, const int* block_tables, int max_pages,
                            const int* seq_first_row, const int* seq_start_pos, int num_seqs, int reach_pages, int nkv, int hd, int page_size,
                            long long num_pages, int window, int* status, cudaStream_t stream) {
    KV4_REQUIRE_SIZES("gb_kv4_expand")
    GB_REQUIRE(dtype == GB_F32 || dtype == GB_BF16, "gb_kv4_expand: unsupported dtype %d", dtype);
    GB_REQUIRE(((uintptr_t)kcache | (uintptr_t)vcache | (uintptr_t)k | (uintptr_t)v) % 16 == 0, "gb_kv4_expand: tensors must be 16-byte aligned");
    GB_REQUIRE(num_seqs >= 0 && num_seqs <= 65535 && max_pages > 0, "gb_kv4_expand: bad batch shape");
    const int pages = reach_pages < max_pages ? reach_pages : max_pages;
    if (num_seqs == 0 || pages <= 0) return 0;
    const dim3 grid(pages, num_seqs), block(KV4_THREADS);
    const unsigned char *kc = (const unsigned char*)kcache, *vc = (const unsigned char*)vcache;
    if (dtype == GB_F32)
        gb_launch(GB_PDL_ELEMENTWISE, kv4_expand_kernel<float>, grid, block, 0, stream, kc, vc, (float*)k, (float*)v, block_tables, max_pages,
                  seq_first_row, seq_start_pos, nkv, hd, page_size, num_pages, window, status);
    else
        gb_launch(GB_PDL_ELEMENTWISE, kv4_expand_kernel<__nv_bfloat16>, grid, block, 0, stream, kc, vc, (__nv_bfloat16*)k, (__nv_bfloat16*)v,
                  block_tables, max_pages, seq_first_row, seq_start_pos, nkv, hd, page_size, num_pages, window, status);
    return gb_check_launch("gb_kv4_expand");
}
