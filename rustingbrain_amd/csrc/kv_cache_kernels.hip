// A paged cache of keys and values: rows written to it, read back from it, and the attention of one new row a sequence over it.
//
// int8 rows have a scale each (per token and head): a = max |x|, scale = a / 127, stored round(127 x / a), ties to even, read back as
// stored * scale.  (127 x is exact for bf16 rows, so one division decides the rounding, and ties are ties.)  A row with an
// infinity or NaN reads back as NaN whole.
//
// All of it is bound by memory (a large copy moves 4.9 TB/s): 23165 bf16 rows of 8 x 128 to 8 bits and back 65 us, 4.4 TB/s (57 where
// the same rows come again, out of the Infinity Cache), f32 rows as they are 180, 4.2 TB/s, to 8 bits 119; new rows over 4 x 131072 cached
// ones, bf16, 8 kv heads of 128, 192 us, 5.6 TB/s; over 64 sequences up to 8192 rows in 8 bits 114 us, 4.3 TB/s (5.0 without the new rows' write and the
// join).  Small calls: launches of 2 to 8 us.
#include "kv_cache_kernels.h"

#include <algorithm>

#include "rbmoe_kernels.h"

namespace rbmoe {

namespace {

typedef uint32_t Any16 __attribute__((ext_vector_type(4), aligned(2), may_alias));

__device__ __forceinline__ unsigned char* cache_block(const CachePool& p, long long page, int head) {
    return p.base + ((size_t)page * p.kv_heads + head) * p.block_bytes();
}
// where element d of row r (within its page) of the values stands, in elements
template <int W, int G>
__device__ __forceinline__ int value_at(int r, int d) {
    return ((r / G) * W + d) * G + r % G;
}

template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&v)[8]) {
    if constexpr (sizeof(T) == 2) {
        const Any16 x = *reinterpret_cast<const Any16*>(p);
        Vec16<T>::widen(make_uint4(x.x, x.y, x.z, x.w), v);
    } else {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const Any16 x = *reinterpret_cast<const Any16*>(p + 4 * i);
            v[4 * i] = __uint_as_float(x.x); v[4 * i + 1] = __uint_as_float(x.y);
            v[4 * i + 2] = __uint_as_float(x.z); v[4 * i + 3] = __uint_as_float(x.w);
        }
    }
}
__device__ __forceinline__ void store8(float* p, const float (&v)[8]) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
        *reinterpret_cast<Any16*>(p + 4 * i) = Any16{__float_as_uint(v[4 * i]), __float_as_uint(v[4 * i + 1]), __float_as_uint(v[4 * i + 2]), __float_as_uint(v[4 * i + 3])};
}
__device__ __forceinline__ void store8(bf16_t* p, const float (&v)[8]) {
    *reinterpret_cast<Any16*>(p) = Any16{pack2(v[0], v[1]), pack2(v[2], v[3]), pack2(v[4], v[5]), pack2(v[6], v[7])};
}
// The 8 values of each of a row's TR threads as bytes, and the scale.  The quotient 127 x / a is rounded as a division would: its approximation by the
// reciprocal is mended by the remainder (Markstein's method: with the correctly rounded reciprocal one step gives the correctly rounded
// quotient), 4 operations where a division takes ten; adding 1.5 * 2^23 rounds to a whole number, ties to even, and leaves it in the low bits.
template <int TR>
__device__ __forceinline__ float quantize(const float (&v)[8], uint2& bytes) {
    uint32_t top = 0;  // of the magnitudes' bits: NaN come out above infinities
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const uint32_t u = __float_as_uint(v[i]) & 0x7fffffffu;
        top = u > top ? u : top;
    }
    top = group_umax(top, TR);
    bytes = make_uint2(0, 0);
    if (top >= 0x7f800000u) return __builtin_nanf("");
    const float most = __uint_as_float(top);
    if (top == 0) return 0.0f;
    const float factor = most > 0x1p100f ? 0x1p-20f : most < 0x1p-100f ? 0x1p60f : 1.0f;  // 127 x and 1 / a stay in range
    const float a = most * factor, r = __fdiv_rn(1.0f, a), n = 127.0f * factor;
    uint32_t q[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float x = n * v[i], y = x * r;
        q[i] = __float_as_uint(__builtin_fmaf(__builtin_fmaf(-y, a, x), r, y) + 12582912.0f);
    }
    auto join = [](uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
        return __builtin_amdgcn_perm(__builtin_amdgcn_perm(d, c, 0x0c0c0400), __builtin_amdgcn_perm(b, a, 0x0c0c0400), 0x05040100);
    };
    bytes = make_uint2(join(q[0], q[1], q[2], q[3]), join(q[4], q[5], q[6], q[7]));
    return __fdiv_rn(most, 127.0f);
}

// A workgroup takes ROWS rows of one head, 8 elements a thread.  Keys go to their places at once; values pass through LDS, where a
// thread picks up a column's elements of neighbouring places: runs of rows in neighbouring places are written in
// pieces of up to 16 bytes.
template <int W>
constexpr int cache_rows() {
    return 16 * (256 / W);
}
// run: how many rows from this one on lie in neighbouring places (a mask of "the next row lies behind this one")
__device__ __forceinline__ int run_from(uint64_t next, int r) {
    const uint64_t stops = ~(next >> r);
    return stops ? (int)__builtin_ctzll(stops) + 1 : 64;
}

// Calls of less than a workgroup a compute unit are bound by the way of a load and a store, not by their number: each element by itself (628 rows of
// 2 x 64 written and read: 8.4 us; by pieces through LDS 10.7).
__device__ __forceinline__ bool few_rows() { return gridDim.x * gridDim.y < 256; }

template <typename T, typename C, int W>
__global__ __launch_bounds__(256) void cache_write_kernel(CacheRows a) {
    constexpr int R = cache_rows<W>(), TR = W / 8, G = 16 / sizeof(C);
    __shared__ __attribute__((aligned(16))) C values[R][W + 16 / sizeof(C)];
    __shared__ long long places[R];
    __shared__ uint64_t neighbours;
    const CachePool& p = a.pool;
    const int head = blockIdx.y, first = blockIdx.x * R, tid = threadIdx.x;
    const long long slots = (long long)p.pages << p.page_shift;
    if (tid < 64) {
        long long at = -1;
        if (tid < R && first + tid < a.rows) at = a.slots[first + tid];
        if (at < 0 || at >= slots) at = -1;
        const long long next = __shfl_down(at, 1);
        const uint64_t mask = __ballot(tid + 1 < R && at >= 0 && next == at + 1);
        if (tid < R) places[tid] = at;
        if (tid == 0) neighbours = mask;
    }
    __syncthreads();
    const int page_mask = (1 << p.page_shift) - 1, c = tid % TR * 8;
    const bool scattered = few_rows() || neighbours == 0;  // (new rows of many sequences: pieces would have one element)
#pragma unroll
    for (int i = 0; i < R * TR / 256; ++i) {
        const int r = i * (256 / TR) + tid / TR;
        if (first + r >= a.rows) break;
        const long long at = places[r];
        float k[8] = {}, v[8] = {};
        if (at >= 0 && c < p.head_dim) {
            load8(static_cast<const T*>(a.k) + (long long)(first + r) * a.k_stride + (long long)head * p.head_dim + c, k);
            load8(static_cast<const T*>(a.v) + (long long)(first + r) * a.v_stride + (long long)head * p.head_dim + c, v);
        }
        unsigned char* const block = cache_block(p, at >= 0 ? at >> p.page_shift : 0, head);
        const int row = (int)(at & page_mask);
        union Stored {  // the 8 values as the cache holds them
            uint2 bytes;
            uint4 words[sizeof(C) == 4 ? 2 : 1];
            C c[8];
        } ks, vs;
        if constexpr (sizeof(C) == 1) {
            const float k_scale = quantize<TR>(k, ks.bytes), v_scale = quantize<TR>(v, vs.bytes);
            if (at >= 0 && tid % TR == 0) {
                float* const scales = reinterpret_cast<float*>(block + 2 * p.half_bytes());
                scales[row] = k_scale;
                scales[(1 << p.page_shift) + row] = v_scale;
            }
        }
        if constexpr (sizeof(C) == 2) {
            ks.words[0] = make_uint4(pack2(k[0], k[1]), pack2(k[2], k[3]), pack2(k[4], k[5]), pack2(k[6], k[7]));
            vs.words[0] = make_uint4(pack2(v[0], v[1]), pack2(v[2], v[3]), pack2(v[4], v[5]), pack2(v[6], v[7]));
        } else if constexpr (sizeof(C) == 4) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                ks.c[j] = k[j];
                vs.c[j] = v[j];
            }
        }
        auto put = [](C* to, const Stored& x) {  // (16-byte boundaries, or 8 for bytes)
            if constexpr (sizeof(C) == 1) *reinterpret_cast<uint2*>(to) = x.bytes;
            else
#pragma unroll
                for (size_t j = 0; j < sizeof(C) / 2; ++j) reinterpret_cast<uint4*>(to)[j] = x.words[j];
        };
        if (at >= 0) put(reinterpret_cast<C*>(block) + (size_t)row * W + c, ks);
        if (!scattered) {
            put(&values[r][c], vs);
        } else if (at >= 0) {
            C* const to = reinterpret_cast<C*>(block + p.half_bytes()) + value_at<W, G>(row, c);
#pragma unroll
            for (int j = 0; j < 8; ++j) to[j * G] = vs.c[j];
        }
    }
    if (scattered) return;
    __syncthreads();
    // column d of 16 rows
    const int d = tid % W, end = tid / W * 16 + 16;
    const uint64_t next = neighbours;
    for (int r = end - 16; r < end;) {
        const long long at = places[r];
        if (at < 0) {
            ++r;
            continue;
        }
        const int row = (int)(at & page_mask), run = min(run_from(next, r), end - r);
        C* const to = reinterpret_cast<C*>(cache_block(p, at >> p.page_shift, head) + p.half_bytes()) + value_at<W, G>(row, d);
        int n = G;
        while (n > 1 && (n > run || (row & (n - 1)))) n >>= 1;
        auto put = [&](auto piece, auto count) {
            typedef decltype(piece) P;
            constexpr int N = decltype(count)::value;
            union {
                P p;
                C c[N];
            } u;
#pragma unroll
            for (int i = 0; i < N; ++i) u.c[i] = values[r + i][d];
            *reinterpret_cast<P*>(to) = u.p;
        };
        constexpr int E = sizeof(C);
        if (n * E == 16) put(uint4{}, std::integral_constant<int, 16 / E>{});
        else if (n * E == 8) put(uint2{}, std::integral_constant<int, 8 / E>{});
        else if (n * E == 4) put(uint32_t{}, std::integral_constant<int, 4 / E>{});
        else if constexpr (E <= 2) {
            if (n * E == 2) put(uint16_t{}, std::integral_constant<int, 2 / E>{});
            else if constexpr (E == 1) put(uint8_t{}, std::integral_constant<int, 1>{});
        }
        r += n;
    }
}

__device__ __forceinline__ void widen8(const float* p, float (&v)[8]) { load8(p, v); }
__device__ __forceinline__ void widen8(const bf16_t* p, float (&v)[8]) { load8(p, v); }
__device__ __forceinline__ void widen8(const int8_t* p, float (&v)[8]) {
    const uint2 w = *reinterpret_cast<const uint2*>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[i] = (float)(int8_t)(w.x >> (8 * i));
        v[4 + i] = (float)(int8_t)(w.y >> (8 * i));
    }
}

// The way back: columns' runs to LDS, then rows.  Rows without a place are zeros.
template <typename T, typename C, int W>
__global__ __launch_bounds__(256) void cache_read_kernel(CacheRows a) {
    constexpr int R = cache_rows<W>(), TR = W / 8, G = 16 / sizeof(C);
    __shared__ __attribute__((aligned(16))) C values[R][W + 16 / sizeof(C)];
    __shared__ long long places[R];
    __shared__ uint64_t neighbours;
    const CachePool& p = a.pool;
    const int head = blockIdx.y, first = blockIdx.x * R, tid = threadIdx.x;
    const long long slots = (long long)p.pages << p.page_shift;
    if (tid < 64) {
        long long at = -1;
        if (tid < R && first + tid < a.rows) at = a.slots[first + tid];
        if (at < 0 || at >= slots) at = -1;
        const long long next = __shfl_down(at, 1);
        const uint64_t mask = __ballot(tid + 1 < R && at >= 0 && next == at + 1);
        if (tid < R) places[tid] = at;
        if (tid == 0) neighbours = mask;
    }
    __syncthreads();
    const int page_mask = (1 << p.page_shift) - 1;
    const bool direct = few_rows();
    const int d = tid % W, end = tid / W * 16 + 16;
    const uint64_t next = neighbours;
    for (int r = direct ? end : end - 16; r < end;) {
        const long long at = places[r];
        if (at < 0) {
            ++r;
            continue;
        }
        const int row = (int)(at & page_mask), run = min(run_from(next, r), end - r);
        const C* const from = reinterpret_cast<const C*>(cache_block(p, at >> p.page_shift, head) + p.half_bytes()) + value_at<W, G>(row, d);
        int n = G;
        while (n > 1 && (n > run || (row & (n - 1)))) n >>= 1;
        auto take = [&](auto piece, auto count) {
            typedef decltype(piece) P;
            constexpr int N = decltype(count)::value;
            union {
                P p;
                C c[N];
            } u;
            u.p = *reinterpret_cast<const P*>(from);
#pragma unroll
            for (int i = 0; i < N; ++i) values[r + i][d] = u.c[i];
        };
        constexpr int E = sizeof(C);
        if (n * E == 16) take(uint4{}, std::integral_constant<int, 16 / E>{});
        else if (n * E == 8) take(uint2{}, std::integral_constant<int, 8 / E>{});
        else if (n * E == 4) take(uint32_t{}, std::integral_constant<int, 4 / E>{});
        else if constexpr (E <= 2) {
            if (n * E == 2) take(uint16_t{}, std::integral_constant<int, 2 / E>{});
            else if constexpr (E == 1) take(uint8_t{}, std::integral_constant<int, 1>{});
        }
        r += n;
    }
    __syncthreads();
    const int c = tid % TR * 8;
    if (c >= p.head_dim) return;
#pragma unroll
    for (int i = 0; i < R * TR / 256; ++i) {
        const int r = i * (256 / TR) + tid / TR;
        if (first + r >= a.rows) continue;
        const long long at = places[r];
        float k[8] = {}, v[8] = {};
        if (at >= 0) {
            const unsigned char* const block = cache_block(p, at >> p.page_shift, head);
            const int row = (int)(at & page_mask);
            widen8(reinterpret_cast<const C*>(block) + (size_t)row * W + c, k);
            if (direct) {
                __attribute__((aligned(16))) C own[8];
                const C* const from = reinterpret_cast<const C*>(block + p.half_bytes()) + value_at<W, G>(row, c);
#pragma unroll
                for (int j = 0; j < 8; ++j) own[j] = from[j * G];
                widen8(own, v);
            } else {
                widen8(&values[r][c], v);
            }
            if constexpr (sizeof(C) == 1) {
                const float* const scales = reinterpret_cast<const float*>(block + 2 * p.half_bytes());
                const float k_scale = scales[row], v_scale = scales[(1 << p.page_shift) + row];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    k[j] *= k_scale;
                    v[j] *= v_scale;
                }
            }
        }
        store8(static_cast<T*>(a.k) + (long long)(first + r) * a.k_stride + (long long)head * p.head_dim + c, k);
        store8(static_cast<T*>(a.v) + (long long)(first + r) * a.v_stride + (long long)head * p.head_dim + c, v);
    }
}

// f(type of the rows, type of the cache, width)
template <typename F>
hipError_t with_types(const CachePool& p, bool bf16_rows, F f) {
    auto wide = [&](auto row, auto cache) -> hipError_t {
        return p.width() == 64 ? f(row, cache, std::integral_constant<int, 64>{}) : f(row, cache, std::integral_constant<int, 128>{});
    };
    if (bf16_rows) return p.dtype == RBMOE_I8 ? wide(bf16_t{}, int8_t{}) : wide(bf16_t{}, bf16_t{});
    return p.dtype == RBMOE_I8 ? wide(float{}, int8_t{}) : wide(float{}, float{});
}

}  // namespace

size_t cache_bytes(const CachePool& p) { return (size_t)p.pages * p.kv_heads * p.block_bytes(); }

hipError_t launch_cache_write(const CacheRows& a, bool bf16_rows, hipStream_t s) {
    return with_types(a.pool, bf16_rows, [&](auto row, auto cache, auto width) {
        constexpr int W = decltype(width)::value, R = cache_rows<W>();
        hipLaunchKernelGGL((cache_write_kernel<decltype(row), decltype(cache), W>), dim3((a.rows + R - 1) / R, a.pool.kv_heads), dim3(256), 0, s, a);
        return hipGetLastError();
    });
}
hipError_t launch_cache_read(const CacheRows& a, bool bf16_rows, hipStream_t s) {
    return with_types(a.pool, bf16_rows, [&](auto row, auto cache, auto width) {
        constexpr int W = decltype(width)::value, R = cache_rows<W>();
        hipLaunchKernelGGL((cache_read_kernel<decltype(row), decltype(cache), W>), dim3((a.rows + R - 1) / R, a.pool.kv_heads), dim3(256), 0, s, a);
        return hipGetLastError();
    });
}

// ---- decode -------------------------------------------------------------------------------------------
//
// A workgroup takes the heads of one group (up to 16) of one sequence over a part of its keys; its waves take tiles of
// keys in turn and load them straight into registers in operand order.  Both products run on the matrix cores: a block
// of 16 keys times the heads' rows (unused columns are zeros: the matrix cores have nothing else to do, the loads decide), then the values' columns
// times the scores.  A tile has four groups of g = 16 / element bytes neighbouring keys, one a row of 16 lanes: key g (m / 4) + 4 b + m % 4 of the
// tile is row m of its block b, so that a lane's scores belong to the g keys whose values it loads as one piece.
// Products of bf16 operands: bf16 and int8 values are such exactly; f32 rows over int8 are cut into three bf16 parts, p (times the
// value's scale) into two for bf16 rows and three for f32 rows: they cost nothing here.  An f32 cache takes the f32 instruction.
template <int N>
__device__ __forceinline__ void cut(const float (&x)[8], bf16x8 (&part)[N]) {
    float rest[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) rest[i] = x[i];
#pragma unroll
    for (int n = 0; n < N; ++n) {
        const uint4 w = make_uint4(pack2(rest[0], rest[1]), pack2(rest[2], rest[3]), pack2(rest[4], rest[5]), pack2(rest[6], rest[7]));
        part[n] = __builtin_bit_cast(bf16x8, w);
        float back[8];
        Vec16<bf16_t>::widen(w, back);
#pragma unroll
        for (int i = 0; i < 8; ++i) rest[i] -= back[i];
    }
}

// p in two parts for values that may hold infinities: both parts are positive where p is, as every part of it times infinity is infinity then.  The first is
// cut off, so that the rest is not negative, and a rest of nothing becomes 2^-24 p, which is below what two parts keep (16 bits).
__device__ __forceinline__ void cut_positive(const float (&x)[8], bf16x8 (&part)[2]) {
    float rest[8];
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 8; ++i) rest[i] = fmaxf(x[i] - __uint_as_float(__float_as_uint(x[i]) & 0xffff0000u), x[i] * 0x1p-24f);
#pragma unroll
    for (int i = 0; i < 4; ++i)  // the upper halves of two
        w[i] = __builtin_amdgcn_perm(__float_as_uint(x[2 * i + 1]), __float_as_uint(x[2 * i]), 0x07060302);
    part[0] = __builtin_bit_cast(bf16x8, make_uint4(w[0], w[1], w[2], w[3]));
    part[1] = __builtin_bit_cast(bf16x8, make_uint4(pack2(rest[0], rest[1]), pack2(rest[2], rest[3]), pack2(rest[4], rest[5]), pack2(rest[6], rest[7])));
}

typedef __attribute__((__vector_size__(4 * sizeof(float)))) float floatx4;

template <typename T, typename C, int W>
struct Decode {
    static constexpr int G = 16 / sizeof(C), KT = 4 * G, NB = G / 4;  // keys of a piece, of a tile; blocks of 16 keys
    static constexpr int KP = W / G / 4;                             // pieces of a key's row that a lane loads
    static constexpr int VP = W / 16;                                // pieces of values (a column each)
    static constexpr int QP = sizeof(C) == 4 ? 1 : sizeof(T) == 4 ? 3 : 1, PP = sizeof(T) == 4 ? 3 : 2;
    struct Keys {
        uint4 k[NB][KP];
        float4 scale[sizeof(C) == 1 ? G / 4 : 1];
    };
    struct Values {
        uint4 v[VP];
        float4 scale[sizeof(C) == 1 ? G / 4 : 1];
    };
};

__device__ __forceinline__ float over_rows_max(float v) {  // over the four rows of 16 lanes
    v = fmaxf(v, __shfl_xor(v, 16));
    return fmaxf(v, __shfl_xor(v, 32));
}
__device__ __forceinline__ float over_rows_sum(float v) {
    v += __shfl_xor(v, 16);
    return v + __shfl_xor(v, 32);
}

// Waves of a workgroup: 4, or as many as registers allow where a call is so small that one workgroup a group of heads takes all of its keys (no
// parts, no second launch).
template <typename C, int W>
constexpr int many_waves() {
    return W == 64 && sizeof(C) != 1 ? 16 : 8;
}
//
// STREAM: the tiles of all sequences, one behind the other, are cut into as many equal ranges as there are workgroups for a group of heads, whatever
// the sequences' lengths are.  A workgroup works off the sequences of its range; it writes rows of those that lie within it, and parts of those that
// pass its ends (number: its own plus the sequence's), which a second launch joins.  Otherwise a workgroup takes one sequence whole.
template <typename C>
constexpr int tile_keys() {
    return 64 / sizeof(C);
}
constexpr int kMostStreamed = 1024;  // sequences: their prefix sums lie in LDS
__device__ __forceinline__ int sequence_length(const DecodeCall& a, int i) {
    return (int)min((long long)min(max(a.lengths[i], 0), a.longest), (long long)a.table_pages << a.pool.page_shift);
}
__device__ __forceinline__ int sequence_tiles(const DecodeCall& a, int i, int keys) {  // (a sequence without keys has one: zeros are written for it)
    return max(1, (sequence_length(a, i) + keys - 1) / keys);
}
__device__ __forceinline__ long long range_start(long long tiles, int i, int n) { return tiles * i / n; }

template <typename T, typename C, int W, int NW, bool STREAM>
__global__ __launch_bounds__(64 * NW, NW == 16 ? 4 : 2) void decode_attention_kernel(DecodeCall a) {
    typedef Decode<T, C, W> X;
    constexpr int G = X::G, KT = X::KT, NB = X::NB, KP = X::KP, VP = X::VP;
    __shared__ float joined[NW][16][W + 4];
    __shared__ float wave_m[NW][16], wave_l[NW][16];
    const CachePool& p = a.pool;
    const int group = a.heads / p.kv_heads, blocks = (group + 15) / 16;
    const int kv = blockIdx.x / blocks, head0 = kv * group + blockIdx.x % blocks * 16, heads = min(16, (kv + 1) * group - head0);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), g = lane >> 4, m16 = lane & 15;
    const int page_mask = (1 << p.page_shift) - 1;

    // the tiles `from` to `to` of a sequence; `part`: where they go if they are not all of it, or -1
    auto work = [&](const int sequence, const int from, const int to, const long long part) {
        const int length = sequence_length(a, sequence);
        const int32_t* const table = a.tables + (long long)sequence * a.table_pages;

        auto entry_at = [&](int t, int quarter) {
            const int i = (t * KT + quarter * G) >> p.page_shift;
            return i < a.table_pages ? table[i] : -1;
        };
        // (under way beside the length and the heads' rows)
        int t = from + wave;
        const int first_k = entry_at(t, m16 >> 2), first_v = entry_at(t, g);

        // the heads' rows as B operand: lane l holds head l % 16
        float q[W / 4];
        bf16x8 qb[sizeof(C) == 4 ? 1 : W / 32][X::QP];
        {
            const T* const row = static_cast<const T*>(a.q) + (long long)sequence * a.q_stride + (long long)(head0 + m16) * p.head_dim;
            const bool there = m16 < heads;
            if constexpr (sizeof(C) == 4) {
#pragma unroll
                for (int c = 0; c < W / 16; ++c) {
                    const int d = 16 * c + 4 * g;
                    Any16 x = {0, 0, 0, 0};
                    if (there && d < p.head_dim) x = *reinterpret_cast<const Any16*>(row + d);
#pragma unroll
                    for (int i = 0; i < 4; ++i) q[4 * c + i] = __uint_as_float(x[i]);
                }
            } else {
#pragma unroll
                for (int c = 0; c < W / 32; ++c) {
                    // bf16 keys: piece 4 c + g of 8; int8: half c % 2 of piece 4 (c / 2) + g of 16
                    const int d = sizeof(C) == 2 ? 32 * c + 8 * g : 64 * (c / 2) + 16 * g + 8 * (c % 2);
                    float x[8] = {};
                    if (there && d < p.head_dim) load8(row + d, x);
                    cut<X::QP>(x, qb[c]);
                }
            }
        }

        // the page of a tile's quarter, or -1: what the table holds there, and whether the quarter has keys
        auto page_of = [&](int entry, int t, int quarter) { return t * KT + quarter * G < length && entry >= 0 && entry < p.pages ? entry : -1; };
        auto entry = [&](int t, int quarter) { return page_of(entry_at(t, quarter), t, quarter); };
        // (a lane loads keys of quarter m16 / 4 and values of quarter g)
        auto load_keys = [&](typename X::Keys& x, int t, int page, int scale_page) {
            const unsigned char* const block = cache_block(p, max(page, 0), kv);
            const int row = ((t * KT + (m16 >> 2) * G) & page_mask) + (m16 & 3);
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int c = 0; c < KP; ++c)
                    x.k[b][c] = *reinterpret_cast<const uint4*>(block + ((size_t)(row + 4 * b) * W + (4 * c + g) * G) * sizeof(C));
            if constexpr (sizeof(C) == 1) {
                const float* const scales = reinterpret_cast<const float*>(cache_block(p, max(scale_page, 0), kv) + 2 * p.half_bytes()) + ((t * KT + g * G) & page_mask);
#pragma unroll
                for (int i = 0; i < G / 4; ++i) x.scale[i] = *reinterpret_cast<const float4*>(scales + 4 * i);
            }
        };
        auto load_values = [&](typename X::Values& x, int t, int page) {
            const unsigned char* const block = cache_block(p, max(page, 0), kv);
            const int row = (t * KT + g * G) & page_mask;
            const unsigned char* const values = block + p.half_bytes() + ((size_t)row * W + m16 * G) * sizeof(C);
#pragma unroll
            for (int c = 0; c < VP; ++c) x.v[c] = *reinterpret_cast<const uint4*>(values + c * 256);
            if constexpr (sizeof(C) == 1) {
                const float* const scales = reinterpret_cast<const float*>(block + 2 * p.half_bytes()) + page_mask + 1 + row;
#pragma unroll
                for (int i = 0; i < G / 4; ++i) x.scale[i] = *reinterpret_cast<const float4*>(scales + 4 * i);
            }
        };

        const float c = a.scale * 1.44269504088896340736f;
        floatx4 acc[VP];
#pragma unroll
        for (int i = 0; i < VP; ++i) acc[i] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
        float m = -__builtin_inff(), l = 0.0f;

        auto score = [&](const typename X::Keys& x, float (&s)[G]) {
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                floatx4 r = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int k = 0; k < KP; ++k) {
                    if constexpr (sizeof(C) == 4) {
                        const float y[4] = {__uint_as_float(x.k[b][k].x), __uint_as_float(x.k[b][k].y), __uint_as_float(x.k[b][k].z), __uint_as_float(x.k[b][k].w)};
#pragma unroll
                        for (int i = 0; i < 4; ++i) r = __builtin_amdgcn_mfma_f32_16x16x4f32(y[i], q[4 * k + i], r, 0, 0, 0);
                    } else if constexpr (sizeof(C) == 2) {
#pragma unroll
                        for (int n = X::QP - 1; n >= 0; --n)
                            r = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, x.k[b][k]), qb[k][n], r, 0, 0, 0);
                    } else {
                        const bf16x8 lo = widen_i8(make_uint2(x.k[b][k].x, x.k[b][k].y)), hi = widen_i8(make_uint2(x.k[b][k].z, x.k[b][k].w));
#pragma unroll
                        for (int n = X::QP - 1; n >= 0; --n) {
                            r = __builtin_amdgcn_mfma_f32_16x16x32_bf16(lo, qb[2 * k][n], r, 0, 0, 0);
                            r = __builtin_amdgcn_mfma_f32_16x16x32_bf16(hi, qb[2 * k + 1][n], r, 0, 0, 0);
                        }
                    }
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) s[4 * b + i] = r[i] * c;
            }
            if constexpr (sizeof(C) == 1) {
#pragma unroll
                for (int i = 0; i < G / 4; ++i) {
                    s[4 * i] *= x.scale[i].x; s[4 * i + 1] *= x.scale[i].y; s[4 * i + 2] *= x.scale[i].z; s[4 * i + 3] *= x.scale[i].w;
                }
            }
        };
        auto add = [&](float (&s)[G], typename X::Values& x, int t, int v_page) {
            // keys behind the end and keys without a page: no score, and nothing of what their values' places hold
            const int left = v_page < 0 ? 0 : length - (t * KT + g * G);
            const bool ragged = __any(left < G);
            if (ragged) {
#pragma unroll
                for (int i = 0; i < G; ++i) s[i] = i < left ? s[i] : -__builtin_inff();
                if constexpr (sizeof(C) != 1) {
                    uint4 keep;
                    uint32_t w[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        w[i] = sizeof(C) == 4 ? (i < left ? ~0u : 0u) : (2 * i < left ? 0xffffu : 0u) | (2 * i + 1 < left ? 0xffff0000u : 0u);
                    keep = make_uint4(w[0], w[1], w[2], w[3]);
#pragma unroll
                    for (int i = 0; i < VP; ++i) {
                        x.v[i].x &= keep.x; x.v[i].y &= keep.y; x.v[i].z &= keep.z; x.v[i].w &= keep.w;
                    }
                }
            }
            float top = s[0];
#pragma unroll
            for (int i = 1; i < G; ++i) top = fmaxf(top, s[i]);
            if (__any(top > m + 8.0f)) {  // (as in the kernels over whole sequences)
                const float next = fmaxf(m, over_rows_max(top)), down = next == m ? 1.0f : __builtin_amdgcn_exp2f(m - next);
                m = next;
                l *= down;
#pragma unroll
                for (int i = 0; i < VP; ++i) acc[i] *= down;
            }
            const float reference = m == -__builtin_inff() ? 0.0f : m;
#pragma unroll
            for (int i = 0; i < G; ++i) {
                s[i] = __builtin_amdgcn_exp2f(s[i] - reference);
                l += s[i];
            }
            if constexpr (sizeof(C) == 4) {
#pragma unroll
                for (int k = 0; k < VP; ++k) {
                    const float y[4] = {__uint_as_float(x.v[k].x), __uint_as_float(x.v[k].y), __uint_as_float(x.v[k].z), __uint_as_float(x.v[k].w)};
#pragma unroll
                    for (int i = 0; i < 4; ++i) acc[k] = __builtin_amdgcn_mfma_f32_16x16x4f32(y[i], s[i], acc[k], 0, 0, 0);
                }
            } else {
                bf16x8 part[G / 8][X::PP];
#pragma unroll
                for (int h = 0; h < G / 8; ++h) {
                    float y[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        y[i] = s[8 * h + i];
                        if constexpr (sizeof(C) == 1) {
                            const float4 f = x.scale[2 * h + i / 4];
                            y[i] = !ragged || 8 * h + i < left ? y[i] * (i % 4 == 0 ? f.x : i % 4 == 1 ? f.y : i % 4 == 2 ? f.z : f.w) : 0.0f;
                        }
                    }
                    if constexpr (sizeof(C) == 2) cut_positive(y, part[h]);
                    else cut<X::PP>(y, part[h]);
                }
#pragma unroll
                for (int k = 0; k < VP; ++k) {
                    if constexpr (sizeof(C) == 2) {
#pragma unroll
                        for (int n = X::PP - 1; n >= 0; --n)
                            acc[k] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, x.v[k]), part[0][n], acc[k], 0, 0, 0);
                    } else {
                        const bf16x8 lo = widen_i8(make_uint2(x.v[k].x, x.v[k].y)), hi = widen_i8(make_uint2(x.v[k].z, x.v[k].w));
#pragma unroll
                        for (int n = X::PP - 1; n >= 0; --n) {
                            acc[k] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(lo, part[0][n], acc[k], 0, 0, 0);
                            acc[k] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(hi, part[1][n], acc[k], 0, 0, 0);
                        }
                    }
                }
            }
        };

        // A tile's values are under way while its scores are made, the next tile's keys while its values are added; page numbers come a tile
        // earlier.  (Behind the last tile that one is loaded again: no load depends on a branch, so that each is waited for alone.)
        if (t < to) {
            typename X::Keys keys;
            typename X::Values values;
            int v_page = page_of(first_v, t, g);
            load_keys(keys, t, page_of(first_k, t, m16 >> 2), v_page);
            int next = min(t + NW, to - 1);
            int k_next = entry(next, m16 >> 2), v_next = entry(next, g);
            for (; t < to; t += NW) {
                load_values(values, t, v_page);
                const int after = min(t + 2 * NW, to - 1);
                const int k_after = entry(after, m16 >> 2), v_after = entry(after, g);
                __builtin_amdgcn_sched_barrier(0);
                float s[G];
                score(keys, s);
                __builtin_amdgcn_sched_barrier(0);
                load_keys(keys, next, k_next, v_next);
                __builtin_amdgcn_sched_barrier(0);
                add(s, values, t, v_page);
                v_page = v_next;
                k_next = k_after;
                v_next = v_after;
                next = after;
            }
        }
        l = over_rows_sum(l);

        // the waves' parts
        if (g == 0) {
            wave_m[wave][m16] = m;
            wave_l[wave][m16] = l;
        }
#pragma unroll
        for (int i = 0; i < VP; ++i)
            *reinterpret_cast<floatx4*>(&joined[wave][m16][16 * i + 4 * g]) = acc[i];
        __syncthreads();
        for (int i = threadIdx.x; i < heads * W; i += 64 * NW) {
            const int h = i / W, d = i % W;
            if (d >= p.head_dim) continue;
            float top = wave_m[0][h];
#pragma unroll
            for (int w = 1; w < NW; ++w) top = fmaxf(top, wave_m[w][h]);
            float o = 0.0f, sum = 0.0f;
#pragma unroll
            for (int w = 0; w < NW; ++w) {
                const float f = wave_m[w][h] == top ? 1.0f : __builtin_amdgcn_exp2f(wave_m[w][h] - top);
                o = __builtin_fmaf(f, joined[w][h][d], o);
                sum = __builtin_fmaf(f, wave_l[w][h], sum);
            }
            if (part < 0) {
                static_cast<T*>(a.out)[((long long)sequence * a.heads + head0 + h) * p.head_dim + d] = from_f32<T>(sum == 0.0f ? 0.0f : o / sum);
            } else {
                const long long row = part * a.heads + head0 + h;
                a.partial[row * W + d] = o;
                if (d == 0) {
                    a.statistics[row * 2] = top;
                    a.statistics[row * 2 + 1] = sum;
                }
            }
        }
    };

    if constexpr (!STREAM) {
        work(blockIdx.y, 0, (sequence_length(a, blockIdx.y) + KT - 1) / KT, -1);
    } else {
        __shared__ long long starts[kMostStreamed + 1], wave_sums[NW];
        constexpr int PER = kMostStreamed / (64 * NW);
        long long own[PER], upto = 0;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int s = threadIdx.x * PER + i;
            own[i] = upto;
            upto += s < a.sequences ? sequence_tiles(a, s, KT) : 0;
        }
        long long before = upto;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const long long y = __shfl_up(before, o);
            before += lane >= o ? y : 0;
        }
        if (lane == 63) wave_sums[wave] = before;
        __syncthreads();
        before -= upto;
        for (int w = 0; w < wave; ++w) before += wave_sums[w];
#pragma unroll
        for (int i = 0; i < PER; ++i) starts[threadIdx.x * PER + i] = before + own[i];
        if (threadIdx.x == 64 * NW - 1) starts[kMostStreamed] = before + upto;
        __syncthreads();
        const long long tiles = starts[kMostStreamed];
        const int ranges = (int)min((long long)gridDim.y, tiles);  // (none without a tile)
        if ((int)blockIdx.y >= ranges) return;
        const long long end = range_start(tiles, blockIdx.y + 1, ranges);
        long long at = range_start(tiles, blockIdx.y, ranges);
        int sequence = 0;  // the last that starts at `at` or before (each has a tile)
        for (int o = kMostStreamed / 2; o > 0; o >>= 1)
            if (sequence + o < a.sequences && starts[sequence + o] <= at) sequence += o;
        for (; at < end; ++sequence) {
            const long long first = starts[sequence], last = starts[sequence + 1], stop = min(end, last);
            work(sequence, (int)(at - first), (int)(stop - first), at == first && stop == last ? -1 : (long long)blockIdx.y + sequence);
            at = stop;
            __syncthreads();  // (the waves' parts have been read)
        }
    }
}

// One workgroup a row whose sequence passes the ends of ranges: its parts.  256 / W threads share a column, each takes every so many parts; their
// sums are added in order.
// Two workgroups a compute unit (1024: 134 us for the 64 sequences above, 512: 124, before loads of the table were moved; in fixed parts of each sequence
// 156); a sequence of 777 rows by one workgroup 10.7 us with its write, in parts 13.0.
constexpr int kDecodeWorkgroups = 512, kLeastPart = 512, kOnePart = 1024;

template <typename T, typename C, int W>
__global__ __launch_bounds__(256) void decode_join_kernel(DecodeCall a) {
    constexpr int S = 256 / W;
    __shared__ float factor[kDecodeWorkgroups], tops[4], columns[S][W], sums[S];
    __shared__ long long wave_sums[2][4];
    const int sequence = blockIdx.x / a.heads, head = blockIdx.x % a.heads, tid = threadIdx.x;
    long long before = 0, tiles = 0;
    for (int i = tid; i < a.sequences; i += 256) {
        const int n = sequence_tiles(a, i, tile_keys<C>());
        tiles += n;
        before += i < sequence ? n : 0;
    }
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        before += __shfl_xor(before, o);
        tiles += __shfl_xor(tiles, o);
    }
    if ((tid & 63) == 0) {
        wave_sums[0][tid >> 6] = before;
        wave_sums[1][tid >> 6] = tiles;
    }
    __syncthreads();
    before = wave_sums[0][0] + wave_sums[0][1] + wave_sums[0][2] + wave_sums[0][3];
    tiles = wave_sums[1][0] + wave_sums[1][1] + wave_sums[1][2] + wave_sums[1][3];
    const int ranges = (int)min((long long)a.ranges, tiles);
    auto range_of = [&](long long tile) {
        int i = (int)(tile * ranges / tiles);
        while (range_start(tiles, i + 1, ranges) <= tile) ++i;
        return i;
    };
    const int first_range = range_of(before), last_range = range_of(before + sequence_tiles(a, sequence, tile_keys<C>()) - 1);
    const int parts = last_range - first_range + 1;
    if (parts == 1) return;  // written already
    // consecutive parts are a.heads rows apart
    const long long row = ((long long)first_range + sequence) * a.heads + head;
    const float* const st = a.statistics + row * 2;
    float top = -__builtin_inff();
    for (int i = tid; i < parts; i += 256) top = fmaxf(top, st[(long long)i * 2 * a.heads]);
    top = group_fmax(top, 64);
    if ((tid & 63) == 0) tops[tid >> 6] = top;
    __syncthreads();
    top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
    for (int i = tid; i < parts; i += 256) {
        const float m = st[(long long)i * 2 * a.heads];
        factor[i] = m == top ? 1.0f : __builtin_amdgcn_exp2f(m - top);
    }
    __syncthreads();
    const int d = tid % W, slice = tid / W;
    const float* const column = a.partial + row * W + d;
    float o = 0.0f, sum = 0.0f;
#pragma unroll 8
    for (int i = slice; i < parts; i += S) {
        o = __builtin_fmaf(factor[i], column[(long long)i * a.heads * W], o);
        sum = __builtin_fmaf(factor[i], st[(long long)i * 2 * a.heads + 1], sum);
    }
    columns[slice][d] = o;
    if (d == 0) sums[slice] = sum;
    __syncthreads();
    if (tid >= a.pool.head_dim) return;
#pragma unroll
    for (int i = 1; i < S; ++i) o += columns[i][tid];
    sum = sums[0];
#pragma unroll
    for (int i = 1; i < S; ++i) sum += sums[i];
    static_cast<T*>(a.out)[((long long)sequence * a.heads + head) * a.pool.head_dim + tid] = from_f32<T>(sum == 0.0f ? 0.0f : o / sum);
}

DecodePlan decode_plan(int sequences, int kv_heads, int group, int longest) {
    const long long groups = (long long)kv_heads * ((group + 15) / 16), rows = groups * sequences;
    if (longest <= kOnePart || sequences > kMostStreamed) return {0, rows <= 256};
    const long long least = ((long long)sequences * longest + kLeastPart - 1) / kLeastPart;
    return {(int)std::max<long long>(1, std::min(kDecodeWorkgroups / groups, least)), false};
}
size_t decode_partials(int sequences, int kv_heads, int group) {  // (ranges + sequences) * heads, of parts that begin or end within a sequence
    return (size_t)kDecodeWorkgroups * std::min(group, 16) + (size_t)std::min(sequences, kMostStreamed) * kv_heads * group;
}

hipError_t launch_decode_attention(const DecodeCall& a, bool bf16_rows, hipStream_t s) {
    const int group = a.heads / a.pool.kv_heads;
    return with_types(a.pool, bf16_rows, [&](auto row, auto cache, auto width) -> hipError_t {
        typedef decltype(row) T;
        typedef decltype(cache) C;
        constexpr int W = decltype(width)::value;
        const int groups = a.pool.kv_heads * ((group + 15) / 16);
        if (a.ranges > 0) hipLaunchKernelGGL((decode_attention_kernel<T, C, W, 4, true>), dim3(groups, a.ranges), dim3(256), 0, s, a);
        else if (a.many) hipLaunchKernelGGL((decode_attention_kernel<T, C, W, many_waves<C, W>(), false>), dim3(groups, a.sequences), dim3(64 * many_waves<C, W>()), 0, s, a);
        else hipLaunchKernelGGL((decode_attention_kernel<T, C, W, 4, false>), dim3(groups, a.sequences), dim3(256), 0, s, a);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess || a.ranges <= 1) return e;
        hipLaunchKernelGGL((decode_join_kernel<T, C, W>), dim3(a.sequences * a.heads), dim3(256), 0, s, a);
        return hipGetLastError();
    });
}

}  // namespace rbmoe
