// Attention of whole sequences with grouped heads, and its backward pass.
//
//   s_ij = scale q_i . k_j   for the keys j that row i sees: j < min(keys, i + keys - queries + 1) (causal), j < keys (not causal)
//   out_i = sum_j p_ij v_j,  p_ij = exp(s_ij - lse_i),  lse_i = log sum_j exp s_ij
//   backward, delta_i = dout_i . out_i:   dp_ij = dout_i . v_j,  ds_ij = p_ij (dp_ij - delta_i)
//   dq_i = scale sum_j ds_ij k_j,   dk_j = scale sum_i ds_ij q_i,   dv_j = sum_i p_ij dout_i   (sums over the heads of a group too)
//
// All products run on the matrix cores in blocks of 32 x 32 x 16 with f32 accumulators: bf16 rows as they are, f32 rows as three bf16 parts.
// A wave owns 32 rows (forward, dq) or 32 keys (dk, dv) and keeps them as the instruction's B operand; the other side goes through LDS in
// tiles, loaded ahead.  A product of two row arrays comes out with the lane's own row in its column and the tile's rows in its registers,
// in the order in which the next product takes them as its B operand: scores never leave registers, and no lane hands a value to another
// except the row statistics.  The second product needs the tile with rows and columns exchanged, which the transposing LDS read gives.  For
// bf16 rows p and ds are rounded to bf16 (the matrix cores take bf16 operands): half a step a term at random, no more than the rounding of the result
// itself, 0.235 % of a gradient in all for 0.166 % (short sequences: in two parts, kShort); their sums, the running maximum and sum of the softmax and all accumulators are f32.  (The sum that
// the forward divides by is that of the unrounded p, which lse needs.  One of the rounded p beside it takes a tenth off what rounding p costs, and 4 to 6 %
// of the time: spilled registers.)
//
// The backward pass takes ds = p (dp - delta) twice, from the queries' side and from the keys', instead of adding one side's sums in
// memory: eight products where five would do, but the same bits from the same call, and no f32 gradients that pass through memory.
//
// Masked places: a masked score is replaced behind the product, whatever it was.  A masked p of zero times an infinity or NaN
// in the tile would still be NaN, so a workgroup that ends with such a value goes over its tiles again: bf16 rows add the blocks
// on the diagonal row by row, f32 rows, whose parts make NaN of an infinity, leave the parts alone (product_f32).  6 x 2048 rows of 8 heads of 64 with
// a NaN in the first value of each: 1.5 ms where clean ones take 0.12; 8192 bf16 rows of 16 heads of 128, backward: 4.9 for 1.5.
//
// What bounds them (a large bf16 product by the library reaches 1370 TFLOP/s, an f32 one 153; times of long calls differ by a tenth from card to card):
//   forward, 16384 rows, 16 heads of 128, bf16, causal: 1.14 to 1.28 ms, 860 to 965 TFLOP/s.  A wave reads every tile from LDS whole, which takes as many
//     cycles of the LDS as the products take of the matrix cores; both are busy seven cycles of ten.
//   heads of 64 (8 x 2048 rows, 8 heads): 52 us, 660 TFLOP/s: a block has half the products and as many exponentials, which take
//     as long as they do; three workgroups a unit instead of two give 8 %.
//   backward, 8192 rows, 16 heads of 128, bf16: 0.59 ms (dq, with its fourth product) and 0.75 (dk, dv), 940 and 730 TFLOP/s of the products taken:
//     registers leave one wave a SIMD, which waits for its exponentials.
//   short or ragged calls: the longest rows' workgroups; f32 rows: 6 products for one, and cutting p and ds in parts.  (Parts rounded to nearest, small
//     products and blocks summed apart: errors of 1.1 to 1.5e-7 of the result forward, 3.3 to 5e-7 of the gradients, where f32 products by the library have
//     2 to 6e-7 and 5e-7 to 1.5e-6.  6 x 2048 rows of 8 heads of 64 117 us, as before with parts cut off; backward of 3 x 700 70 for 67.  Heads of 128: 4096
//     rows of 16 heads 457 us, 150 TFLOP/s.)
#include "attention_kernels.h"

#include <algorithm>
#include <atomic>
#include <type_traits>

#include "rbmoe_kernels.h"

namespace rbmoe {

namespace {

constexpr int kThreads = 256, kWaves = 4;
constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.693147180559945309417f;

// What is loaded for rows and columns that are not there.  (A branch around the load would do too, but not in kernels that fill their registers: at the
// end of a region that only some lanes run, the compiler may save a register before the others are back, and theirs is lost.)
__device__ __attribute__((aligned(16))) uint32_t zero_piece[8];
template <typename T>
__device__ __forceinline__ const T* or_zeros(const T* p, bool there) {
    return there ? p : reinterpret_cast<const T*>(zero_piece);
}

typedef uint32_t Any16 __attribute__((ext_vector_type(4), aligned(2), may_alias));
typedef uint32_t Any8 __attribute__((ext_vector_type(2), aligned(2), may_alias));
typedef short v4i16 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) v4i16 lds_v4i16;

__device__ __forceinline__ uint32_t lds_address(const char* p) {
    return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const char*)p;
}
// 64 lanes' 16 bytes to consecutive LDS addresses (the same in all lanes) without registers on the way
__device__ __forceinline__ void issue_dma(uint32_t lds_addr, const void* src) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" : : "s"(lds_addr), "v"(src) : "memory");
}

__device__ __forceinline__ void issue_dma_word(uint32_t lds_addr, const void* src) {  // and their 4 bytes
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" : : "s"(lds_addr), "v"(src) : "memory");
}

__device__ __forceinline__ float other_half_max(float v) {
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float other_half_sum(float v) {
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// ---- operands ------------------------------------------------------------------------------------
// f32 rows as matrix operands: three bf16 parts of 8 bits each, each the rest of those in front rounded to nearest, which add up to the value exactly.
// Of the nine products of two values' parts the six largest are taken; the others are below 2^-25 of the product and of any sign.
// (32 x 32 x 16 of them take 192 cycles, the f32 instruction 512.)  An infinity's rest is NaN, and so is what it goes into, which the workgroup
// notices, as it does values that round to one (above 3.39e38).
struct Parts8 {
    bf16x8 part[3];
};
__device__ __forceinline__ Parts8 cut8(const float (&x)[8]) {
    Parts8 r;
    float rest[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) rest[i] = x[i];
#pragma unroll
    for (int n = 0; n < 3; ++n) {
        const uint4 w = make_uint4(pack2(rest[0], rest[1]), pack2(rest[2], rest[3]), pack2(rest[4], rest[5]), pack2(rest[6], rest[7]));
        r.part[n] = __builtin_bit_cast(bf16x8, w);
        if (n == 2) break;
        float back[8];
        Vec16<bf16_t>::widen(w, back);
#pragma unroll
        for (int i = 0; i < 8; ++i) rest[i] -= back[i];
    }
    return r;
}

template <typename T>
struct Mma;
template <>
struct Mma<bf16_t> {
    static constexpr int P = 1;  // parts
    typedef bf16x8 Rows;         // 8 elements of a row
    struct Cols {                // a 32 x 32 block of scores as the second product takes it
        bf16x8 c[2];
    };
    static __device__ __forceinline__ bf16x8 part(const Rows& r, int) { return r; }
    static __device__ __forceinline__ bf16x8 part(const Cols& p, int k, int) { return p.c[k]; }
    static __device__ __forceinline__ Cols cols(const floatx16& p) {
        Cols r;
#pragma unroll
        for (int i = 0; i < 2; ++i)
            r.c[i] = __builtin_bit_cast(bf16x8, make_uint4(pack2(p[8 * i], p[8 * i + 1]), pack2(p[8 * i + 2], p[8 * i + 3]),
                                                           pack2(p[8 * i + 4], p[8 * i + 5]), pack2(p[8 * i + 6], p[8 * i + 7])));
        return r;
    }
    static __device__ __forceinline__ Cols rest(const floatx16& p, const Cols& rounded) {  // what rounding left, rounded
        floatx16 r;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            float back[8];
            Vec16<bf16_t>::widen(__builtin_bit_cast(uint4, rounded.c[i]), back);
#pragma unroll
            for (int j = 0; j < 8; ++j) r[8 * i + j] = p[8 * i + j] - back[j];
        }
        return cols(r);
    }
    static __device__ __forceinline__ float total(const Cols& p, float sum) {  // of the lane's own values
        typedef __attribute__((__vector_size__(2 * sizeof(__bf16)))) __bf16 bf16x2;
        const bf16x2 one = {(__bf16)1.0f, (__bf16)1.0f};
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint4 w = __builtin_bit_cast(uint4, p.c[i]);
            sum = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, w.x), one, sum, false);
            sum = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, w.y), one, sum, false);
            sum = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, w.z), one, sum, false);
            sum = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, w.w), one, sum, false);
        }
        return sum;
    }
    static __device__ __forceinline__ float rounded(float v) { return bf16_bits_to_f32(f32_to_bf16_bits(v)); }
    // exp of x / `unit`: scores and references are kept times log2 e, for the base-2 exponential
    static constexpr float unit = kLog2e, natural = kLn2;
    static __device__ __forceinline__ float exponential(float x) { return __builtin_amdgcn_exp2f(x); }
};
template <>
struct Mma<float> {
    static constexpr int P = 3;
    typedef Parts8 Rows;
    struct Cols {
        Parts8 c[2];
    };
    static __device__ __forceinline__ bf16x8 part(const Rows& r, int i) { return r.part[i]; }
    static __device__ __forceinline__ bf16x8 part(const Cols& p, int k, int i) { return p.c[k].part[i]; }
    static __device__ __forceinline__ Cols cols(const floatx16& p) {
        Cols r;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const float x[8] = {p[8 * k], p[8 * k + 1], p[8 * k + 2], p[8 * k + 3], p[8 * k + 4], p[8 * k + 5], p[8 * k + 6], p[8 * k + 7]};
            r.c[k] = cut8(x);
        }
        return r;
    }
    static __device__ __forceinline__ float rounded(float v) { return v; }
    // (the factor is the caller's scale as it is, and only the difference is rounded with log2 e)
    static constexpr float unit = 1.0f, natural = 1.0f;
    static __device__ __forceinline__ float exponential(float x) { return __builtin_amdgcn_exp2f(x * kLog2e); }
};
template <typename T>
using RowsOf = typename Mma<T>::Rows;

__device__ __forceinline__ void load8(const bf16_t* p, float (&v)[8]) {
    const Any16 x = *reinterpret_cast<const Any16*>(p);
    Vec16<bf16_t>::widen(make_uint4(x.x, x.y, x.z, x.w), v);
}
__device__ __forceinline__ void load8(const float* p, float (&v)[8]) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const Any16 x = *reinterpret_cast<const Any16*>(p + 4 * i);
        v[4 * i] = __uint_as_float(x.x); v[4 * i + 1] = __uint_as_float(x.y); v[4 * i + 2] = __uint_as_float(x.z); v[4 * i + 3] = __uint_as_float(x.w);
    }
}

// ---- a tile of rows in LDS ---------------------------------------------------------------------
// N rows of D elements as bf16 parts, one part behind the other, without padding, in 16-byte pieces; piece c of row r lies at place c ^ swizzle(r), so
// that the reads along rows (eight rows, one piece) and the transposing reads (four rows, 32 bytes) both find their banks free.
template <typename T, int D, int N>
struct Tile {
    static constexpr int P = Mma<T>::P, CH = D / 8, ROW = D * 2, PART = N * ROW, BYTES = P * PART;
    static constexpr int KC = D / 16;  // steps of a product along D: each takes two pieces of a row, one per half of the wave
    static constexpr int DB = D / 32;  // blocks of 32 columns
    static __device__ __forceinline__ int swizzle(int r) {
        if constexpr (CH == 8) return ((r >> 1) & 1) << 2 | ((r >> 2) & 3);
        return (r & 3) << 2 | ((r >> 2) & 3);
    }
    static __device__ __forceinline__ const char* piece(const char* tile, int r, int c) { return tile + r * ROW + ((c ^ swizzle(r)) << 4); }
    static __device__ __forceinline__ void quad(const char* tile, int r, int d, float (&y)[4]) {  // (of bf16 rows)
        const uint2 x = *reinterpret_cast<const uint2*>(piece(tile, r, d / 8) + d % 8 * 2);
        y[0] = __uint_as_float(x.x << 16); y[1] = __uint_as_float(x.x & 0xffff0000u);
        y[2] = __uint_as_float(x.y << 16); y[3] = __uint_as_float(x.y & 0xffff0000u);
    }

    // The rows from `first` on of a sequence's n, by TEAM waves; columns from head_dim on and rows from n on are zeros.  begin() has the loads
    // under way, finish() leaves them in the tile: bf16 rows on 16-byte boundaries get there without it.
    template <int TEAM, bool A>
    struct Stager {
        static constexpr int UNITS = N * CH / (64 * TEAM);  // pieces of 8 elements a lane
        float x[P == 3 ? UNITS : 1][8];
        Any16 raw[P == 1 && !A ? UNITS : 1];
        __device__ __forceinline__ void begin(char* tile, const T* __restrict__ base, long long stride, int first, int n, int pieces) {
            const int wave = TEAM == 1 ? 0 : __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), lane = threadIdx.x & 63;
#pragma unroll
            for (int i = 0; i < UNITS; ++i) {
                const int at = (i * TEAM + wave) * 64, p = at + lane, r = p / CH, c = (p % CH) ^ swizzle(r);
                const bool there = first + r < n && c < pieces;
                const T* const src = base + (long long)(first + r) * stride + c * 8;
                if constexpr (P == 3) {
                    load8(or_zeros(src, there), x[i]);
                } else if constexpr (A) {
                    issue_dma(lds_address(tile) + at * 16, or_zeros(src, there));
                } else {
                    raw[i] = *reinterpret_cast<const Any16*>(or_zeros(src, there));
                }
            }
        }
        __device__ __forceinline__ void finish(char* tile) {
            if constexpr (P == 3 || !A) {
#pragma unroll
                for (int i = 0; i < UNITS; ++i) {
                    char* const to = tile + (i * TEAM * 64 + (int)(threadIdx.x & (64 * TEAM - 1))) * 16;
                    if constexpr (P == 3) {
                        const Parts8 parts = cut8(x[i]);
#pragma unroll
                        for (int k = 0; k < 3; ++k) *reinterpret_cast<bf16x8*>(to + k * PART) = parts.part[k];
                    } else {
                        *reinterpret_cast<uint4*>(to) = make_uint4(raw[i].x, raw[i].y, raw[i].z, raw[i].w);
                    }
                }
            }
        }
    };

    // The product of 32 of the tile's rows with the wave's own: register i of lane l holds tile row 8 (i / 4) + 4 (l / 32) + i % 4, own row l % 32.
    static __device__ __forceinline__ floatx16 product(const char* tile, int row0, const RowsOf<T> (&own)[KC]) {
        const int lane = threadIdx.x & 63;
        floatx16 c, small;  // (sums of their own: the large one is rounded once a step, not six times)
#pragma unroll
        for (int i = 0; i < 16; ++i) c[i] = small[i] = 0.0f;
#pragma unroll
        for (int kc = 0; kc < KC; ++kc) {
            bf16x8 rows[P];
#pragma unroll
            for (int i = 0; i < P; ++i) rows[i] = *reinterpret_cast<const bf16x8*>(piece(tile + i * PART, row0 + (lane & 31), 2 * kc + (lane >> 5)));
#pragma unroll
            for (int s = P - 1; s > 0; --s)
#pragma unroll
                for (int i = 0; i <= s; ++i) small = __builtin_amdgcn_mfma_f32_32x32x16_bf16(rows[i], Mma<T>::part(own[kc], s - i), small, 0, 0, 0);
            c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(rows[0], Mma<T>::part(own[kc], 0), c, 0, 0, 0);
        }
        if constexpr (P > 1)
#pragma unroll
            for (int i = 0; i < 16; ++i) c[i] += small[i];
        return c;
    }
    // acc[d][own] += sum over the block's 32 rows r of tile[r][d] p[r][own]; of M's parts (bf16_t: the first ones alone).  Several products a term are
    // summed up over the block first, so that the sum over all blocks is rounded once a block.
    template <typename M = T>
    static __device__ __forceinline__ void add(floatx16 (&acc)[DB], const char* tile, int row0, const typename Mma<M>::Cols& p) {
        constexpr int P = Mma<M>::P;
        const int lane = threadIdx.x & 63, h = lane >> 5, j = (lane >> 2) & 3;
        const int c0 = 2 * ((lane >> 4) & 1) + ((lane >> 1) & 1), in = (lane & 1) * 8;
        auto columns = [&](int k, int b, int part) {
            const int r = row0 + 16 * k + 4 * h + j;
            union {
                v4i16 x[2];
                bf16x8 v;
            } u;
            u.x[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4i16*)(piece(tile + part * PART, r, 4 * b + c0) + in));
            u.x[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4i16*)(piece(tile + part * PART, r + 8, 4 * b + c0) + in));
            return u.v;
        };
        if constexpr (P == 1) {
#pragma unroll
            for (int k = 0; k < 2; ++k)
#pragma unroll
                for (int b = 0; b < DB; ++b)
                    acc[b] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(columns(k, b, 0), Mma<M>::part(p, k, 0), acc[b], 0, 0, 0);
        } else {
#pragma unroll
            for (int b = 0; b < DB; ++b) {
                floatx16 c;
#pragma unroll
                for (int i = 0; i < 16; ++i) c[i] = 0.0f;
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    bf16x8 cols[P];
#pragma unroll
                    for (int i = 0; i < P; ++i) cols[i] = columns(k, b, i);
#pragma unroll
                    for (int s = P - 1; s >= 0; --s)  // small ones first
#pragma unroll
                        for (int i = 0; i <= s; ++i) c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(cols[i], Mma<M>::part(p, k, s - i), c, 0, 0, 0);
                }
#pragma unroll
                for (int i = 0; i < 16; ++i) acc[b][i] += c[i];
            }
        }
    }
};
__device__ __forceinline__ int block_row(int i) { return 8 * (i >> 2) + 4 * ((threadIdx.x >> 5) & 1) + (i & 3); }

// Tile::add one element after the other: for a block of which some places are masked, whatever the tile holds there.  Row by row, the places that
// `sees`(row) allows; `quad`(row, d, y) gives four elements of a row.
template <typename T, int D, typename Q, typename F>
__device__ __forceinline__ void add_seen(floatx16 (&acc)[D / 32], const floatx16& p, Q quad, F sees) {
    const int lane = threadIdx.x & 63, h = lane >> 5;
#pragma clang loop unroll(disable)
    for (int r = 0; r < 32; ++r) {
        float x = 0.0f;
#pragma unroll
        for (int i = 0; i < 16; ++i) x = i == (r >> 3) * 4 + (r & 3) ? p[i] : x;
        x = Mma<T>::rounded(__shfl(x, (lane & 31) + 32 * ((r >> 2) & 1)));
        const bool seen = sees(r);
#pragma unroll
        for (int b = 0; b < D / 32; ++b)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                float y[4] = {};
                quad(r, 32 * b + 8 * e + 4 * h, y);
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[b][4 * e + j] = seen ? __builtin_fmaf(x, y[j], acc[b][4 * e + j]) : acc[b][4 * e + j];
            }
    }
}
// Parts of an infinity do not multiply as it does (0 times infinity, infinity minus infinity), so a pass over f32 rows that hold one takes
// them as they are, from memory: the scores by the f32 instruction, in the same order and layout as Tile::product, sums by add_seen.
template <int D, typename T>
__device__ __forceinline__ floatx16 product_f32(const T* __restrict__ rows, long long stride, int n, const T* __restrict__ own, bool there, int pieces) {
    const int lane = threadIdx.x & 63, h = lane >> 5;
    floatx16 c;
#pragma unroll
    for (int i = 0; i < 16; ++i) c[i] = 0.0f;
#pragma clang loop unroll(disable)
    for (int kc = 0; kc < D / 16; ++kc) {
        float x[8], y[8];
        load8(or_zeros(rows + (long long)(lane & 31) * stride + (2 * kc + h) * 8, (lane & 31) < n && 2 * kc + h < pieces), x);
        load8(or_zeros(own + (2 * kc + h) * 8, there && 2 * kc + h < pieces), y);
#pragma unroll
        for (int i = 0; i < 8; ++i) c = __builtin_amdgcn_mfma_f32_32x32x2f32(x[i], y[i], c, 0, 0, 0);
    }
    return c;
}
// `quad` of add_seen over n rows in memory
template <typename T>
__device__ __forceinline__ auto quads_of(const T* __restrict__ rows, long long stride, int n, int head_dim) {
    return [=](int r, int d, float (&y)[4]) {
        const Any16 x = *reinterpret_cast<const Any16*>(or_zeros(rows + (long long)r * stride + d, r < n && d < head_dim));
#pragma unroll
        for (int j = 0; j < 4; ++j) y[j] = __uint_as_float(x[j]);
    };
}
template <int N>
__device__ __forceinline__ bool any_not_finite(const floatx16 (&acc)[N]) {
    bool bad = false;
#pragma unroll
    for (int b = 0; b < N; ++b)
#pragma unroll
        for (int i = 0; i < 16; ++i) bad |= !(fabsf(acc[b][i]) < __builtin_inff());
    return bad;
}

// ---- a wave's own rows ---------------------------------------------------------------------------
// The row of lane l % 32 as the products' B operand, zeros where it or its columns are not there.
template <typename T, int D>
__device__ __forceinline__ void load_own(const T* __restrict__ row, bool there, int pieces, RowsOf<T> (&own)[D / 16]) {
    const int h = (threadIdx.x >> 5) & 1;
#pragma unroll
    for (int kc = 0; kc < D / 16; ++kc) {
        const bool in = there && 2 * kc + h < pieces;
        if constexpr (sizeof(T) == 4) {
            float x[8];
            load8(or_zeros(row + (2 * kc + h) * 8, in), x);
            own[kc] = cut8(x);
        } else {
            const Any16 x = *reinterpret_cast<const Any16*>(or_zeros(row + (2 * kc + h) * 8, in));
            own[kc] = __builtin_bit_cast(bf16x8, x);
        }
    }
    // In use here and now: the wait for these loads would otherwise stand in front of their first use in the loop over tiles, where every turn
    // would wait for the next tile's loads with it.
    if constexpr (sizeof(T) == 2)
#pragma unroll
        for (int kc = 0; kc < D / 16; ++kc) asm volatile("" : "+v"(own[kc]));
}
__device__ __forceinline__ void store4(float* p, float a, float b, float c, float d) {
    *reinterpret_cast<Any16*>(p) = Any16{__float_as_uint(a), __float_as_uint(b), __float_as_uint(c), __float_as_uint(d)};
}
__device__ __forceinline__ void store4(bf16_t* p, float a, float b, float c, float d) {
    *reinterpret_cast<Any8*>(p) = Any8{pack2(a, b), pack2(c, d)};
}
// acc[d][own] of lane l's own row to `row`, times `factor`.  TEAM 1: the sum over the workgroup's four waves, in their order, each of which stores a
// quarter; all threads call, `room` is 4 x D x 128 bytes of LDS that nobody reads any more.
template <typename T, int D, int TEAM>
__device__ __forceinline__ void store_own(const floatx16 (&acc)[D / 32], T* row, bool there, float factor, int head_dim, char* room) {
    const int lane = threadIdx.x & 63, h = lane >> 5;
    if constexpr (TEAM == 1) {
        const int wave = threadIdx.x >> 6;
        float4* const parts = reinterpret_cast<float4*>(room) + lane;
#pragma unroll
        for (int b = 0; b < D / 32; ++b)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                parts[((wave * (D / 32) + b) * 4 + e) * 64] = make_float4(acc[b][4 * e], acc[b][4 * e + 1], acc[b][4 * e + 2], acc[b][4 * e + 3]);
        __syncthreads();
#pragma unroll
        for (int b = 0; b < D / 32; ++b) {
            float x[4] = {};
#pragma unroll
            for (int w = 0; w < kWaves; ++w) {
                const float4 y = parts[((w * (D / 32) + b) * 4 + wave) * 64];
                x[0] += y.x; x[1] += y.y; x[2] += y.z; x[3] += y.w;
            }
            const int d = 32 * b + 8 * wave + 4 * h;
            if (there && d < head_dim) store4(row + d, x[0] * factor, x[1] * factor, x[2] * factor, x[3] * factor);
        }
        __syncthreads();
    } else {
        if (!there) return;
#pragma unroll
        for (int b = 0; b < D / 32; ++b)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int d = 32 * b + 8 * e + 4 * h;
                if (d < head_dim) store4(row + d, acc[b][4 * e] * factor, acc[b][4 * e + 1] * factor, acc[b][4 * e + 2] * factor, acc[b][4 * e + 3] * factor);
            }
    }
}
// The sum (or maximum) of a lane's value over the four waves; all threads call.
template <bool MAX>
__device__ __forceinline__ float over_waves(float v, char* room) {
    float* const parts = reinterpret_cast<float*>(room);
    parts[threadIdx.x] = v;
    __syncthreads();
    const float x[kWaves] = {parts[threadIdx.x & 63], parts[64 + (threadIdx.x & 63)], parts[128 + (threadIdx.x & 63)], parts[192 + (threadIdx.x & 63)]};
    __syncthreads();
    return MAX ? fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])) : (x[0] + x[1]) + (x[2] + x[3]);
}

// ---- sequences -------------------------------------------------------------------------------------
__device__ __forceinline__ Sequence sequence_of(const AttentionCall& a, int i) {
    return cut_sequence(a.query_begin[i], a.query_count[i], a.key_begin[i], a.key_count[i], a.query_rows, a.key_rows, a.longest_queries, a.longest_keys);
}
// Which tile, head and sequence a workgroup takes.  Workgroup i runs on XCD i % 8: where the heads divide among them, every XCD has
// its own heads (neighbours, so that a group's heads share their keys in one L2), otherwise all take turns.  Tiles in descending order: the last are the
// longest where later rows see more keys.
struct Place {
    int tile, head, sequence;
};
__device__ __forceinline__ Place place_of(int heads, int sequences, int tiles, bool descending) {
    int i = blockIdx.x;
    Place p;
    if (heads % 8 == 0) {
        const int per = heads / 8, xcd = i & 7;
        i >>= 3;
        p.head = xcd * per + i % per;
        i /= per;
    } else {
        p.head = i % heads;
        i /= heads;
    }
    p.sequence = i % sequences;
    p.tile = i / sequences;
    if (descending) p.tile = tiles - 1 - p.tile;
    return p;
}

// How a workgroup's four waves share the work.  TEAM 4: each owns 32 rows, the tiles are common.  TEAM 1: all own the same 32 rows, each takes every
// fourth tile, stages it for itself, and their sums are added at the end: four times the workgroups, for calls that have few.
// A tile has 64 rows where the rest leaves registers for two blocks' operands on their way, 32 otherwise (grad_q, 8 sequences up to 2048 rows, 8 heads of
// 64: 60 us by 32, 77 by 64; 8192 rows, 16 heads of 128: 700 and 650).
template <typename T, int D, int TEAM, bool GRAD_Q = false>
constexpr int tile_rows() {
    return sizeof(T) == 2 && TEAM == 4 && !(GRAD_Q && D == 64) ? 64 : 32;
}
// Stages of tiles.  TEAM 4: two, one is filled while the other is used.  TEAM 1: one, where workgroups beside this one on its compute unit are busy
// meanwhile, or the next tile waits in registers; two for kernels whose registers leave room for one workgroup (ALONE).  (us with one / two, bf16: heads of 64,
// backward of 8 sequences up to 2048 rows 158 / 161, of 512 rows 22.8 / 22.9, forward of 2048 rows 17.1 / 16.2; heads of 128, backward of 8192 rows 1356 / 1338.)
template <typename T, int D, int TEAM, bool ALONE>
constexpr int tile_stages() {
    return TEAM == 4 || (ALONE && sizeof(T) == 2 && D == 128) ? 2 : 1;
}
template <typename T, int D, int TEAM, int N, bool ALONE>
constexpr int tiles_lds(int extra) {  // of two tiles of N rows and `extra` bytes a stage
    return (kWaves / TEAM) * tile_stages<T, D, TEAM, ALONE>() * (2 * Tile<T, D, N>::BYTES + extra);
}
// bf16 sequences of so few rows or keys take p and ds in two parts for the gradients, 16 bits: a few roundings decide there and do not even out (sequences of two
// rows were up to 0.3 % off, 1.9 times the rounding of the result).  For all sequences it would be 0.166 % instead of 0.235, and a quarter of the time more:
// 8192 rows of 16 heads of 128 1.68 ms for 1.34, 8 x 2048 of 8 heads of 64 195 us for 158.
constexpr int kShort = 32;
__device__ __forceinline__ bool few_terms(const Sequence& s) { return min(s.nq, s.nk) <= kShort; }

__device__ __forceinline__ void wait_for_tile(bool common) {
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");  // this wave's part of the tile has landed, its reads of the other stage are done
    if (common) __syncthreads();                                 // and the other waves'
}

// A wave's or workgroup's tiles from `start` to `end`, `step` apart: the next one's loads are under way while one is used.  With one stage
// f32 rows wait in registers meanwhile; bf16 rows, which are loaded straight into it, are waited for.
template <int STAGES, int PARTS, int TEAM, typename B, typename F, typename U>
__device__ __forceinline__ void over_tiles(int start, int end, int step, B begin, F finish, U use) {
    if constexpr (STAGES == 1 && PARTS == 1) {
        for (int t = start; t < end; t += step) {
            wait_for_tile(false);
            begin(0, t);
            finish(0);
            wait_for_tile(false);
            use(0, t);
        }
    } else {
        if (start < end) {
            begin(0, start);
            finish(0);
        }
        for (int t = start, buf = 0; t < end; t += step, buf ^= STAGES - 1) {
            wait_for_tile(TEAM == 4);
            const bool more = t + step < end;
            if (more) begin(buf ^ (STAGES - 1), t + step);
            use(buf, t);
            if (more) finish(buf ^ (STAGES - 1));
        }
    }
}

// ---- forward ----------------------------------------------------------------------------------------

template <typename T, int D, int TEAM, bool A>
__global__ __launch_bounds__(kThreads, D * sizeof(T) > 256 || (sizeof(T) == 4 && TEAM == 1) ? 1 : D * sizeof(T) == 128 ? 3 : 2) void attention_forward_kernel(AttentionCall a) {
    constexpr int N = tile_rows<T, D, TEAM>(), NB = N / 32, OWN = 32 * TEAM, STAGES = tile_stages<T, D, TEAM, false>();
    typedef Tile<T, D, N> Tl;
    constexpr int BYTES = Tl::BYTES;
    extern __shared__ __attribute__((aligned(16))) char attention_lds[];  // two stages of keys and values
    const int tiles = (a.most_queries + OWN - 1) / OWN;
    const Place at = place_of(a.heads, a.sequences, tiles, a.causal);
    const Sequence s = sequence_of(a, at.sequence);
    const int first = at.tile * OWN;
    if (first >= s.nq) return;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), h = lane >> 5;
    const int kv = at.head / (a.heads / a.kv_heads), pieces = a.head_dim / 8;
    const T* const k = static_cast<const T*>(a.k) + (long long)s.k0 * a.k_stride + (long long)kv * a.head_dim;
    const T* const v = static_cast<const T*>(a.v) + (long long)s.k0 * a.v_stride + (long long)kv * a.head_dim;
    const int wave_first = TEAM == 1 ? first : first + 32 * wave, row = wave_first + (lane & 31);
    const bool there = row < s.nq;
    const T* const q_row = static_cast<const T*>(a.q) + (long long)(s.q0 + row) * a.q_stride + (long long)at.head * a.head_dim;
    RowsOf<T> q[Tl::KC];
    load_own<T, D>(q_row, there, pieces, q);

    // the keys that a row sees are those below its limit
    auto limit = [&](int r) { return a.causal ? min(max(r + s.ahead + 1, 0), s.nk) : s.nk; };
    const int own_limit = limit(row), least = limit(wave_first), most = limit(min(wave_first + 31, s.nq - 1));
    const int end = limit(min(first + OWN, s.nq) - 1);
    constexpr int STEP = TEAM == 1 ? kWaves * N : N;
    const int start = TEAM == 1 ? wave * N : 0;
    char* const tiles_at = attention_lds + (TEAM == 1 ? wave * STAGES * 2 * BYTES : 0);
    const float c = a.scale * Mma<T>::unit;
    floatx16 acc[Tl::DB];
    float m, l;

    auto pass = [&](auto careful) {
        constexpr bool F32 = decltype(careful)::value && sizeof(T) == 4;
#pragma unroll
        for (int b = 0; b < Tl::DB; ++b)
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[b][i] = 0.0f;
        m = -__builtin_inff();
        l = 0.0f;
        typename Tl::template Stager<TEAM, A> keys, values;
        auto begin = [&](int buf, int t) {
            char* const to = tiles_at + buf * 2 * BYTES;
            keys.begin(to, k, a.k_stride, t, s.nk, pieces);
            values.begin(to + BYTES, v, a.v_stride, t, s.nk, pieces);
        };
        auto finish = [&](int buf) {
            char* const to = tiles_at + buf * 2 * BYTES;
            keys.finish(to);
            values.finish(to + BYTES);
        };
        auto use = [&](int buf, int t) {
            if (t >= most || wave_first >= s.nq) return;
            const char* const kt = tiles_at + buf * 2 * BYTES;
            const char* const vt = kt + BYTES;
            floatx16 p[NB];
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                const int r0 = t + 32 * b;
                if constexpr (F32) p[b] = product_f32<D>(k + (long long)r0 * a.k_stride, a.k_stride, s.nk - r0, q_row, there, pieces);
                else p[b] = Tl::product(kt, 32 * b, q);
            }
            if (t + N > least) {
#pragma unroll
                for (int b = 0; b < NB; ++b)
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        if (t + 32 * b + block_row(i) >= own_limit) p[b][i] = -__builtin_inff();
            }
            // The exponents' arguments by the reference that there is: it moves only when a score passes it by 2^8 (f32 rows: e^8).  The results are
            // the same, sums and accumulators have room for it, and after a few tiles nothing has to be scaled.
            const float reference = m == -__builtin_inff() ? 0.0f : m;
            float top = -__builtin_inff();
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    p[b][i] = __builtin_fmaf(p[b][i], c, -reference);
                    top = fmaxf(top, p[b][i]);
                }
            if (__any(top > (m == -__builtin_inff() ? m : 8.0f))) {
                top = other_half_max(top);
                const float next = top > (m == -__builtin_inff() ? m : 0.0f) ? reference + top : m;
                const float down = next == m ? 1.0f : Mma<T>::exponential(m - next), shift = next == m ? 0.0f : next - reference;
                m = next;
                l *= down;
#pragma unroll
                for (int b = 0; b < Tl::DB; ++b)
#pragma unroll
                    for (int i = 0; i < 16; ++i) acc[b][i] *= down;
#pragma unroll
                for (int b = 0; b < NB; ++b)
#pragma unroll
                    for (int i = 0; i < 16; ++i) p[b][i] -= shift;
            }
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                float sum = 0.0f;  // of the block: the sum over all is rounded once a block
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    p[b][i] = Mma<T>::exponential(p[b][i]);
                    sum += p[b][i];
                }
                l += sum;
            }
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                const int r0 = t + 32 * b;
                auto sees = [&](int r) { return r0 + r < own_limit; };
                if constexpr (F32) {
                    add_seen<T, D>(acc, p[b], quads_of(v + (long long)r0 * a.v_stride, a.v_stride, s.nk - r0, a.head_dim), sees);
                } else if (decltype(careful)::value && t + N > least) {
                    add_seen<T, D>(acc, p[b], [&](int r, int d, float (&y)[4]) { Tl::quad(vt, 32 * b + r, d, y); }, sees);
                } else {
                    Tl::add(acc, vt, 32 * b, Mma<T>::cols(p[b]));
                }
            }
        };
        over_tiles<STAGES, Tl::P, TEAM>(start, end, STEP, begin, finish, use);
    };
    pass(std::false_type{});
    if (__syncthreads_or(any_not_finite(acc))) pass(std::true_type{});

    l = other_half_sum(l);
    if constexpr (TEAM == 1) {  // to one reference
        __syncthreads();
        const float all = over_waves<true>(m, attention_lds), down = m == all ? 1.0f : Mma<T>::exponential(m - all);
        m = all;
        l = over_waves<false>(l * down, attention_lds);
#pragma unroll
        for (int b = 0; b < Tl::DB; ++b)
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[b][i] *= down;
    }
    const long long to = (long long)(s.q0 + row) * a.heads + at.head;
    store_own<T, D, TEAM>(acc, static_cast<T*>(a.out) + to * a.head_dim, there, l == 0.0f ? 0.0f : 1.0f / l, a.head_dim, attention_lds);
    if (there && a.lse && h == 0 && (TEAM == 4 || wave == 0))
        a.lse[(long long)at.head * a.query_rows + s.q0 + row] =
            l == 0.0f ? -__builtin_inff() : (m == -__builtin_inff() ? 0.0f : m * Mma<T>::natural) + __builtin_amdgcn_logf(l) * kLn2;
}

// ---- backward: gradients of the queries ------------------------------------------------------------------
template <typename T, int D, int TEAM, bool A>
__global__ __launch_bounds__(kThreads, D == 128 || sizeof(T) == 4 ? 1 : 2) void attention_grad_q_kernel(AttentionCall a) {
    constexpr int N = tile_rows<T, D, TEAM, true>(), NB = N / 32, OWN = 32 * TEAM, STAGES = tile_stages<T, D, TEAM, true>();
    typedef Tile<T, D, N> Tl;
    constexpr int BYTES = Tl::BYTES;
    extern __shared__ __attribute__((aligned(16))) char attention_lds[];
    const int tiles = (a.most_queries + OWN - 1) / OWN;
    const Place at = place_of(a.heads, a.sequences, tiles, a.causal);
    const Sequence s = sequence_of(a, at.sequence);
    const int first = at.tile * OWN;
    if (first >= s.nq) return;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), h = lane >> 5;
    const int kv = at.head / (a.heads / a.kv_heads), pieces = a.head_dim / 8;
    const T* const k = static_cast<const T*>(a.k) + (long long)s.k0 * a.k_stride + (long long)kv * a.head_dim;
    const T* const v = static_cast<const T*>(a.v) + (long long)s.k0 * a.v_stride + (long long)kv * a.head_dim;
    const int wave_first = TEAM == 1 ? first : first + 32 * wave, row = wave_first + (lane & 31);
    const bool there = row < s.nq;
    const long long in_out = ((long long)(s.q0 + row) * a.heads + at.head) * a.head_dim, in_lse = (long long)at.head * a.query_rows + s.q0 + row;
    const T* const q_row = static_cast<const T*>(a.q) + (long long)(s.q0 + row) * a.q_stride + (long long)at.head * a.head_dim;
    const T* const dout_row = static_cast<const T*>(a.grad_out) + in_out;
    RowsOf<T> q[Tl::KC], dout[Tl::KC];
    load_own<T, D>(q_row, there, pieces, q);
    load_own<T, D>(dout_row, there, pieces, dout);

    float delta = 0.0f;
#pragma unroll
    for (int kc = 0; kc < Tl::KC; ++kc) {
        const bool in = there && 2 * kc + h < pieces;
        float x[8], y[8];
        load8(or_zeros(static_cast<const T*>(a.out) + in_out + (2 * kc + h) * 8, in), x);
        load8(or_zeros(dout_row + (2 * kc + h) * 8, in), y);
#pragma unroll
        for (int i = 0; i < 8; ++i) delta = __builtin_fmaf(x[i], y[i], delta);
    }
    delta = other_half_sum(delta);
    float reference = *or_zeros(a.lse + in_lse, there) * Mma<T>::unit;
    asm volatile("" : "+v"(reference));  // (as in load_own)

    auto limit = [&](int r) { return a.causal ? min(max(r + s.ahead + 1, 0), s.nk) : s.nk; };
    const int own_limit = limit(row), least = limit(wave_first), most = limit(min(wave_first + 31, s.nq - 1));
    const int end = limit(min(first + OWN, s.nq) - 1);
    constexpr int STEP = TEAM == 1 ? kWaves * N : N;
    const int start = TEAM == 1 ? wave * N : 0;
    char* const tiles_at = attention_lds + (TEAM == 1 ? wave * STAGES * 2 * BYTES : 0);
    const float c = a.scale * Mma<T>::unit;
    // delta comes from `out` as it was stored, and ds is rounded for bf16 rows.  Both errors make a row's ds add up to something
    // else than its true sum of zero, and where keys share a direction that goes along it.  So the sum of the ds is taken
    // off again in proportion to p (grad_q -= sum * mean key; the sum is small, bf16 does for the mean), and delta handed on as what makes the
    // sum of the unrounded ones zero.
    floatx16 acc[Tl::DB], mean[Tl::DB];
    float sum, rounded_sum;

    auto pass = [&](auto careful) {
        constexpr bool F32 = decltype(careful)::value && sizeof(T) == 4;
#pragma unroll
        for (int b = 0; b < Tl::DB; ++b)
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[b][i] = mean[b][i] = 0.0f;
        sum = rounded_sum = 0.0f;
        typename Tl::template Stager<TEAM, A> keys, values;
        auto begin = [&](int buf, int t) {
            char* const to = tiles_at + buf * 2 * BYTES;
            keys.begin(to, k, a.k_stride, t, s.nk, pieces);
            values.begin(to + BYTES, v, a.v_stride, t, s.nk, pieces);
        };
        auto finish = [&](int buf) {
            char* const to = tiles_at + buf * 2 * BYTES;
            keys.finish(to);
            values.finish(to + BYTES);
        };
        auto use = [&](int buf, int t) {
            if (t >= most || wave_first >= s.nq) return;
            const char* const kt = tiles_at + buf * 2 * BYTES;
            const char* const vt = kt + BYTES;
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                const int r0 = t + 32 * b;
                floatx16 p, dp;
                if constexpr (F32) {
                    p = product_f32<D>(k + (long long)r0 * a.k_stride, a.k_stride, s.nk - r0, q_row, there, pieces);
                    dp = product_f32<D>(v + (long long)r0 * a.v_stride, a.v_stride, s.nk - r0, dout_row, there, pieces);
                } else {
                    p = Tl::product(kt, 32 * b, q);
                    dp = Tl::product(vt, 32 * b, dout);
                }
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    p[i] = Mma<T>::exponential(__builtin_fmaf(p[i], c, -reference));
                    dp[i] = p[i] * (dp[i] - delta);
                }
                if (t + N > least) {
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        if (r0 + block_row(i) >= own_limit) p[i] = dp[i] = 0.0f;
                }
                const auto ds = Mma<T>::cols(dp);
#pragma unroll
                for (int i = 0; i < 16; ++i) sum += dp[i];
                if constexpr (sizeof(T) == 2) {
                    rounded_sum = Mma<T>::total(ds, rounded_sum);
                    if (!decltype(careful)::value && few_terms(s)) {
                        const auto rest = Mma<T>::rest(dp, ds);
                        rounded_sum = Mma<T>::total(rest, rounded_sum);
                        Tl::add(acc, kt, 32 * b, rest);
                    }
                }
                auto sees = [&](int r) { return r0 + r < own_limit; };
                if constexpr (F32) {
                    auto quad = quads_of(k + (long long)r0 * a.k_stride, a.k_stride, s.nk - r0, a.head_dim);
                    add_seen<T, D>(acc, dp, quad, sees);
                    add_seen<T, D>(mean, p, quad, sees);
                } else if (decltype(careful)::value && t + N > least) {
                    auto quad = [&](int r, int d, float (&y)[4]) { Tl::quad(kt, 32 * b + r, d, y); };
                    add_seen<T, D>(acc, dp, quad, sees);
                    add_seen<T, D>(mean, p, quad, sees);
                } else {
                    Tl::add(acc, kt, 32 * b, ds);
                    Tl::template add<bf16_t>(mean, kt, 32 * b, Mma<bf16_t>::cols(p));
                }
            }
        };
        over_tiles<STAGES, Tl::P, TEAM>(start, end, STEP, begin, finish, use);
    };
    pass(std::false_type{});
    if (__syncthreads_or(any_not_finite(acc))) pass(std::true_type{});
    if constexpr (TEAM == 1) __syncthreads();
    if constexpr (sizeof(T) == 4) rounded_sum = sum;
    rounded_sum = other_half_sum(rounded_sum);
    sum = other_half_sum(sum);
    if constexpr (TEAM == 1) {
        rounded_sum = over_waves<false>(rounded_sum, attention_lds);
        sum = over_waves<false>(sum, attention_lds);
    }
    delta += sum;
#pragma unroll
    for (int b = 0; b < Tl::DB; ++b)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[b][i] = __builtin_fmaf(-rounded_sum, mean[b][i], acc[b][i]);
    if (there && h == 0 && (TEAM == 4 || wave == 0)) {
        a.delta[in_lse] = reference;
        a.delta[(long long)a.heads * a.query_rows + in_lse] = delta;
    }
    // (a row that sees one key has p = 1 and ds = 0, whatever the roundings made of it)
    store_own<T, D, TEAM>(acc, static_cast<T*>(a.grad_q) + (long long)(s.q0 + row) * a.q_stride + (long long)at.head * a.head_dim, there,
                          own_limit == 1 ? 0.0f : a.scale, a.head_dim, attention_lds);
}

// ---- backward: gradients of keys and values -------------------------------------------------------------
template <typename T, int D, int TEAM, bool A>
__global__ __launch_bounds__(kThreads, D == 128 || sizeof(T) == 4 ? 1 : 2) void attention_grad_kv_kernel(AttentionCall a) {
    constexpr int N = tile_rows<T, D, TEAM>(), NB = N / 32, OWN = 32 * TEAM, STAGES = tile_stages<T, D, TEAM, true>();
    typedef Tile<T, D, N> Tl;
    constexpr int BYTES = Tl::BYTES, STAGE = 2 * BYTES + 2 * N * 4;
    extern __shared__ __attribute__((aligned(16))) char attention_lds[];  // two stages of queries, gradients, lse and delta
    const int tiles = (a.most_keys + OWN - 1) / OWN;
    const Place at = place_of(a.kv_heads * a.shares, a.sequences, tiles, false);
    const Sequence s = sequence_of(a, at.sequence);
    const int first = at.tile * OWN, kv = at.head / a.shares, share = at.head % a.shares;
    const int group = a.heads / a.kv_heads / a.shares, head0 = at.head * group;  // the heads of this share of the group
    if (first >= s.nk) return;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int pieces = a.head_dim / 8;
    const int wave_first = TEAM == 1 ? first : first + 32 * wave, key = wave_first + (lane & 31);
    const bool there = key < s.nk;
    RowsOf<T> k[Tl::KC], v[Tl::KC];
    const T* const k_row = static_cast<const T*>(a.k) + (long long)(s.k0 + key) * a.k_stride + (long long)kv * a.head_dim;
    const T* const v_row = static_cast<const T*>(a.v) + (long long)(s.k0 + key) * a.v_stride + (long long)kv * a.head_dim;
    load_own<T, D>(k_row, there, pieces, k);
    load_own<T, D>(v_row, there, pieces, v);

    // the rows that see a key are those from its start on
    auto start = [&](int j) { return a.causal ? max(j - s.ahead, 0) : 0; };
    const int lone = a.causal ? -s.ahead : -1;  // the row that sees one key: p = 1 and ds = 0
    const int own_start = start(key), least = start(wave_first), most = start(wave_first + 31);
    const int begin = start(first) / N * N, turns = begin < s.nq ? (s.nq - begin + N - 1) / N : 0, all = turns * group;
    constexpr int STEP = TEAM == 1 ? kWaves : 1;
    const int mine = TEAM == 1 ? wave : 0;
    char* const tiles_at = attention_lds + (TEAM == 1 ? wave * STAGES * STAGE : 0);
    const float c = a.scale * Mma<T>::unit;
    const long long dout_stride = (long long)a.heads * a.head_dim;
    auto q_of = [&](int head) { return static_cast<const T*>(a.q) + (long long)s.q0 * a.q_stride + (long long)head * a.head_dim; };
    auto dout_of = [&](int head) { return static_cast<const T*>(a.grad_out) + s.q0 * dout_stride + (long long)head * a.head_dim; };
    floatx16 dk[Tl::DB], dv[Tl::DB];

    auto pass = [&](auto careful) {
        constexpr bool F32 = decltype(careful)::value && sizeof(T) == 4;
#pragma unroll
        for (int b = 0; b < Tl::DB; ++b)
#pragma unroll
            for (int i = 0; i < 16; ++i) dk[b][i] = dv[b][i] = 0.0f;
        // turn i: head i / turns of the group, rows from begin + N (i % turns) on
        typename Tl::template Stager<TEAM, A> queries, gradients;
        float statistic = 0.0f;
        auto begin_tile = [&](int buf, int i) {
            const int head = head0 + i / turns, t = begin + i % turns * N;
            char* const to = tiles_at + buf * STAGE;
            if (TEAM == 1 || wave < 2 * N / 64) {  // references, then deltas
                const int at = TEAM == 1 ? lane : threadIdx.x, r = t + at % N;
                const float* const from = a.delta + (at < N ? 0 : (long long)a.heads * a.query_rows) + (long long)head * a.query_rows + s.q0 + r;
                if constexpr (Tl::P == 3) statistic = *or_zeros(from, r < s.nq);
                else issue_dma_word(lds_address(to) + 2 * BYTES + (TEAM == 1 ? 0 : wave * 256), or_zeros(from, r < s.nq));
            }
            queries.begin(to, q_of(head), a.q_stride, t, s.nq, pieces);
            gradients.begin(to + BYTES, dout_of(head), dout_stride, t, s.nq, pieces);
        };
        auto finish = [&](int buf) {
            char* const to = tiles_at + buf * STAGE;
            if constexpr (Tl::P == 3)
                if (TEAM == 1 || wave < 2 * N / 64) *reinterpret_cast<float*>(to + 2 * BYTES + (TEAM == 1 ? lane : threadIdx.x) * 4) = statistic;
            queries.finish(to);
            gradients.finish(to + BYTES);
        };
        auto use = [&](int buf, int i) {
            const int head = head0 + i / turns, t = begin + i % turns * N;
            if (t + N <= least || wave_first >= s.nk) return;
            const char* const qt = tiles_at + buf * STAGE;
            const char* const ot = qt + BYTES;
            const float* const references = reinterpret_cast<const float*>(ot + BYTES);
            const bool masked = t < most || t + N > s.nq;
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                const int r0 = t + 32 * b;
                floatx16 p, dp;
                if constexpr (F32) {
                    p = product_f32<D>(q_of(head) + r0 * a.q_stride, a.q_stride, s.nq - r0, k_row, there, pieces);
                    dp = product_f32<D>(dout_of(head) + r0 * dout_stride, dout_stride, s.nq - r0, v_row, there, pieces);
                } else {
                    p = Tl::product(qt, 32 * b, k);
                    dp = Tl::product(ot, 32 * b, v);
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int r = 32 * b + block_row(4 * e);
                    const float4 x = *reinterpret_cast<const float4*>(references + r), y = *reinterpret_cast<const float4*>(references + N + r);
                    const float xs[4] = {x.x, x.y, x.z, x.w}, ys[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        p[4 * e + j] = Mma<T>::exponential(__builtin_fmaf(p[4 * e + j], c, -xs[j]));
                        dp[4 * e + j] = p[4 * e + j] * (dp[4 * e + j] - ys[j]);
                    }
                }
                auto sees = [&](int r) { return r0 + r >= own_start && r0 + r < s.nq; };
                if (masked) {
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        if (!sees(block_row(e))) p[e] = dp[e] = 0.0f;
                        if (r0 + block_row(e) == lone) dp[e] = 0.0f;
                    }
                }
                if constexpr (F32) {
                    add_seen<T, D>(dv, p, quads_of(dout_of(head) + r0 * dout_stride, dout_stride, s.nq - r0, a.head_dim), sees);
                    add_seen<T, D>(dk, dp, quads_of(q_of(head) + r0 * a.q_stride, a.q_stride, s.nq - r0, a.head_dim), sees);
                } else if (decltype(careful)::value && masked) {
                    add_seen<T, D>(dv, p, [&](int r, int d, float (&y)[4]) { Tl::quad(ot, 32 * b + r, d, y); }, sees);
                    add_seen<T, D>(dk, dp, [&](int r, int d, float (&y)[4]) { Tl::quad(qt, 32 * b + r, d, y); }, sees);
                } else {
                    const auto ps = Mma<T>::cols(p), ds = Mma<T>::cols(dp);
                    Tl::add(dv, ot, 32 * b, ps);
                    Tl::add(dk, qt, 32 * b, ds);
                    if constexpr (sizeof(T) == 2)
                        if (!decltype(careful)::value && few_terms(s)) {
                            Tl::add(dv, ot, 32 * b, Mma<T>::rest(p, ps));
                            Tl::add(dk, qt, 32 * b, Mma<T>::rest(dp, ds));
                        }
                }
            }
        };
        over_tiles<STAGES, Tl::P, TEAM>(mine, all, STEP, begin_tile, finish, use);
    };
    pass(std::false_type{});
    if (__syncthreads_or(any_not_finite(dk) || any_not_finite(dv))) pass(std::true_type{});
    if constexpr (TEAM == 1) __syncthreads();
    const float factor = s.nk == 1 ? 0.0f : 1.0f;
    if (a.shares == 1) {
        store_own<T, D, TEAM>(dk, static_cast<T*>(a.grad_k) + (long long)(s.k0 + key) * a.k_stride + (long long)kv * a.head_dim, there, factor * a.scale,
                              a.head_dim, attention_lds);
        store_own<T, D, TEAM>(dv, static_cast<T*>(a.grad_v) + (long long)(s.k0 + key) * a.v_stride + (long long)kv * a.head_dim, there, 1.0f, a.head_dim,
                              attention_lds);
    } else {
        float* const part = a.parts + (((long long)share * a.key_rows + s.k0 + key) * a.kv_heads + kv) * 2 * a.head_dim;
        store_own<float, D, TEAM>(dk, part, there, factor, a.head_dim, attention_lds);
        store_own<float, D, TEAM>(dv, part + a.head_dim, there, 1.0f, a.head_dim, attention_lds);
    }
}

// The shares' sums, in their order; four elements a thread.
template <typename T>
__global__ __launch_bounds__(kThreads) void attention_add_shares_kernel(AttentionCall a) {
    const Sequence s = sequence_of(a, blockIdx.y);
    const int quads = a.head_dim / 4, i = blockIdx.x * kThreads + threadIdx.x;
    const int d = i % quads * 4, kv = i / quads % a.kv_heads, row = i / quads / a.kv_heads;
    if (row >= s.nk) return;
    const float* part = a.parts + ((long long)(s.k0 + row) * a.kv_heads + kv) * 2 * a.head_dim + d;
    float k[4] = {}, v[4] = {};
    for (int n = 0; n < a.shares; ++n, part += (long long)a.key_rows * a.kv_heads * 2 * a.head_dim)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            k[j] += part[j];
            v[j] += part[a.head_dim + j];
        }
    store4(static_cast<T*>(a.grad_k) + (long long)(s.k0 + row) * a.k_stride + (long long)kv * a.head_dim + d, k[0] * a.scale, k[1] * a.scale, k[2] * a.scale, k[3] * a.scale);
    store4(static_cast<T*>(a.grad_v) + (long long)(s.k0 + row) * a.v_stride + (long long)kv * a.head_dim + d, v[0], v[1], v[2], v[3]);
}

bool whole_pieces(const void* p, long long stride, int size) {
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && stride * size % 16 == 0;
}

// f(element type, padded head width, waves a team, rows on 16-byte boundaries, where that matters)
template <typename F>
hipError_t with_kernel(bool bf16, int head_dim, bool few, bool aligned, F f) {
    auto rows = [&](auto type, auto width, auto team) -> hipError_t {
        if constexpr (sizeof(type) == 2)
            if (aligned) return f(type, width, team, std::true_type{});
        return f(type, width, team, std::false_type{});
    };
    auto team = [&](auto type, auto width) -> hipError_t {
        if constexpr (sizeof(type) * decltype(width)::value > 256)  // (four teams' tiles of three parts are more than the LDS)
            return rows(type, width, std::integral_constant<int, 4>{});
        else return few ? rows(type, width, std::integral_constant<int, 1>{}) : rows(type, width, std::integral_constant<int, 4>{});
    };
    auto width = [&](auto type) -> hipError_t {
        return head_dim <= 64 ? team(type, std::integral_constant<int, 64>{}) : team(type, std::integral_constant<int, 128>{});
    };
    return bf16 ? width(bf16_t{}) : width(float{});
}

// Workgroups of 128 rows below which 32 rows make one.  Two of them fill a compute unit, so 512 fill the device.  us with teams of 1 / 4: 5 bf16 prompts
// behind 4000 keys, 32 heads of 128 (800 workgroups) 188 / 147; keys' gradients of 8 sequences up to 2048 rows, 2 kv heads of 64 (256) 92 / 190.
constexpr int kFew = 512;
// Workgroups of 32 keys below which a group's heads get their own (half as many for heads of 128, which leave room for one workgroup a unit).  us of the
// backward pass with / without: 8 heads of 64 in groups of 4, bf16: 2 x 2048 rows (256 workgroups) 76 / 97, 1 x 512 23 / 31, 8 x 512 (256, short ones) 46 / 43;
// f32: 4 x 1024 193 / 224.  Heads of 128 in groups of 4: 1 x 512 (64) bf16 35 / 45, f32 193 / 451; 1 x 1024 (128) bf16 65 / 82; 1 x 64 of 32 heads (16) 24 / 22, where the
// third launch shows.
constexpr int kShared = 512;
// Whether a launch over `longest` rows of `heads` heads a sequence would have few workgroups of 128 rows.
bool few_workgroups(const AttentionCall& a, int longest, int heads) { return (long long)((longest + 127) / 128) * heads * a.sequences < kFew; }

template <typename K>
hipError_t launch(K kernel, std::atomic<unsigned long long>& once, const AttentionCall& a, int tiles, int heads, int lds, hipStream_t s) {
    const hipError_t e = once_per_device(once, [&] {
        return hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, lds);
    });
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(kernel, dim3((unsigned)tiles * heads * a.sequences), dim3(kThreads), lds, s, a);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_attention_forward(const AttentionCall& a, bool bf16, hipStream_t s) {
    const int size = bf16 ? 2 : 4;
    const bool aligned = whole_pieces(a.k, a.k_stride, size) && whole_pieces(a.v, a.v_stride, size);
    return with_kernel(bf16, a.head_dim, few_workgroups(a, a.most_queries, a.heads), aligned, [&](auto type, auto width, auto team, auto whole) {
        typedef decltype(type) T;
        constexpr int D = decltype(width)::value, TEAM = decltype(team)::value, OWN = 32 * TEAM;
        static std::atomic<unsigned long long> once{0};
        return launch(attention_forward_kernel<T, D, TEAM, decltype(whole)::value>, once, a, (a.most_queries + OWN - 1) / OWN, a.heads,
                      tiles_lds<T, D, TEAM, tile_rows<T, D, TEAM>(), false>(0), s);
    });
}

hipError_t launch_attention_backward(const AttentionCall& a, bool bf16, hipStream_t s) {
    const int size = bf16 ? 2 : 4;
    hipError_t e = hipSuccess;
    if (a.most_queries > 0) {
        const bool aligned = whole_pieces(a.k, a.k_stride, size) && whole_pieces(a.v, a.v_stride, size);
        e = with_kernel(bf16, a.head_dim, few_workgroups(a, a.most_queries, a.heads), aligned, [&](auto type, auto width, auto team, auto whole) {
            typedef decltype(type) T;
            constexpr int D = decltype(width)::value, TEAM = decltype(team)::value, OWN = 32 * TEAM;
            static std::atomic<unsigned long long> once{0};
            return launch(attention_grad_q_kernel<T, D, TEAM, decltype(whole)::value>, once, a, (a.most_queries + OWN - 1) / OWN, a.heads,
                          tiles_lds<T, D, TEAM, tile_rows<T, D, TEAM, true>(), true>(0), s);
        });
    }
    if (e != hipSuccess || a.most_keys == 0) return e;
    // A kv head's workgroups go through all heads of its group.  Where they are few, each head gets workgroups of its own, and their sums are added.
    AttentionCall b = a;
    const int group = a.heads / a.kv_heads;
    const long long blocks = (long long)((a.most_keys + 31) / 32) * a.kv_heads * a.sequences;
    const bool few = few_workgroups(a, a.most_keys, a.kv_heads);
    b.shares = few && group > 1 && blocks < (a.head_dim <= 64 ? kShared : kShared / 2) && (long long)a.key_rows * a.kv_heads <= a.part_rows ? group : 1;
    const bool aligned = whole_pieces(a.q, a.q_stride, size) && whole_pieces(a.grad_out, a.head_dim, size);
    e = with_kernel(bf16, a.head_dim, few, aligned, [&](auto type, auto width, auto team, auto whole) {
        typedef decltype(type) T;
        constexpr int D = decltype(width)::value, TEAM = decltype(team)::value, OWN = 32 * TEAM;
        static std::atomic<unsigned long long> once{0};
        return launch(attention_grad_kv_kernel<T, D, TEAM, decltype(whole)::value>, once, b, (a.most_keys + OWN - 1) / OWN, a.kv_heads * b.shares,
                      tiles_lds<T, D, TEAM, tile_rows<T, D, TEAM>(), true>(8 * tile_rows<T, D, TEAM>()), s);
    });
    if (e != hipSuccess || b.shares == 1) return e;
    const dim3 grid((unsigned)(((long long)a.most_keys * a.kv_heads * a.head_dim / 4 + kThreads - 1) / kThreads), a.sequences);
    if (bf16) hipLaunchKernelGGL(attention_add_shares_kernel<bf16_t>, grid, dim3(kThreads), 0, s, b);
    else hipLaunchKernelGGL(attention_add_shares_kernel<float>, grid, dim3(kThreads), 0, s, b);
    return hipGetLastError();
}

int attention_part_rows(int backward_rows, int kv_heads, int group) {
    return group == 1 ? 0 : (int)std::min<long long>((long long)backward_rows * kv_heads, kShared * 32);
}

}  // namespace rbmoe
