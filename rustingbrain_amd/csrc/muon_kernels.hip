// Orthogonalised updates: the quintic Newton-Schulz iteration on the matrix cores, and the optimiser step around it.
//
//   X0 = U / (|U|_F + 1e-7)                                  [m, n] with m <= n: a taller matrix is taken transposed
//   A = X X^T,  B = a I + b A + c A A,  X <- B X             (a, b, c) = (3.4445, -4.7750, 2.0315), `steps` times
//
// acts on the singular values alone, p(s) = a s + b s^3 + c s^5: p maps [0, 1.2025] into itself, and five steps bring everything from
// 0.003 up into [0.68, 1.21].  So throughout |X| <= 1.21, |A| <= 1.47 and |B| <= a (spectral norms, which bound the elements).
//
// Precision.  The result is f32-grade: every operand is kept as two fp16 numbers, hi = fp16(2^14 v) and lo = fp16(2^14 v - hi), together 22
// bits.  The bounds above keep 2^14 v below 65504.  lo ends at fp16's 2^-24, so the 22 bits are whole from |v| = 2^-16 up and the error is 2^-39
// below: next to an |X|_F of about one that is 2^-39 sqrt(m n) at most, 2^-28 for 1408 x 1408.  A matrix whose |U|_F is not far above
// 1e-7 begins with a smaller |X|_F, |U|_F / (|U|_F + 1e-7), and grows by 3.4 a step at most: such an X is kept times a power of two (Lift) that
// brings it near one at every step.  A and B need none: their errors count beside a.  A product is three on the matrix
// cores, hi hi + hi lo + lo hi, with f32 sums; what is left out is 2^-22 of a term.  That is three fp16 products at 16 times the rate of
// the f32 ones.  (Two bf16 parts hold 16 bits, and five steps of them end 1e-5 from the exact result where f32 ends 2e-6.)
//
// What bounds it.  Large stacks: 128 x [704, 1024] f32 takes 4.8 ms a step, 0.46 of them the passes over gradients, momentum and weights
// at the rate of a copy.  The rest is 3.6 TFLOP of fp16 multiplies (A and B counted by halves), 0.83 PFLOP/s where a large fp16 product of
// the library reaches 1.08: a launch without its output runs at 1.25 over all the blocks that its tiles cover, and the blocks below
// the diagonal and the output (0.74 GB for X, 0.25 for A and for B) take the difference.  Small ones: every launch starts on cold second-level caches and
// writes its output through at the end, 3 to 6 us for 17 launches (1 x [512, 512] 79 us).
//
// Layout.  Operands lie in the order in which the matrix cores take them: a fragment is 32 rows x 16 columns of the reduction, lane l
// holds row l % 32, columns 8 (l / 32) .. + 7, so 64 lanes x 16 bytes hold the hi parts of a fragment and the 1024 bytes behind them
// the lo parts.  Every load of an operand is then 1 KB of neighbouring bytes.  Rows and columns are padded to 32 with zeros, which
// stay zero through every step.  X is kept both ways, X [m rows, n reduced] for A and X^T [n rows, m reduced] for B X.
#include "muon_kernels.h"

#include <algorithm>

namespace rbmoe {

namespace {

constexpr float kA = 3.4445f, kB = -4.7750f, kC = 2.0315f;
constexpr float kUp = 16384.0f, kDown = 1.0f / 16384.0f;  // 2^14
constexpr int kFragment = 2048;                           // bytes: hi, then lo
constexpr int kRawBuffer = 0x00020000;                    // descriptor word 3: untyped, no swizzle
constexpr int kVolatile = (int)0x80000000u;               // of a buffer load: not to be moved

typedef __attribute__((__vector_size__(8 * sizeof(_Float16)))) _Float16 halfx8;
typedef __attribute__((__vector_size__(4 * sizeof(_Float16)))) _Float16 halfx4;
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ void split(float scaled, _Float16& hi, _Float16& lo) {
    hi = (_Float16)scaled;
    lo = (_Float16)(scaled - (float)hi);
}

// Sizes of the operands of one matrix.
struct Shape {
    int m, n;            // m <= n
    int mg, ng;          // groups of 32
    __host__ __device__ size_t x_bytes() const { return (size_t)mg * ng * 2 * kFragment; }  // X, X^T
    __host__ __device__ size_t a_bytes() const { return (size_t)mg * mg * 2 * kFragment; }  // A, B
};
Shape shape_of(int rows, int cols) {
    Shape s;
    s.m = std::min(rows, cols);
    s.n = std::max(rows, cols);
    s.mg = (s.m + 31) / 32;
    s.ng = (s.n + 31) / 32;
    return s;
}

// ---- momentum and |U|^2 ----------------------------------------------------------------------------
constexpr int kNormElements = 4096;  // of one workgroup
int norm_parts(int rows, int cols) { return (int)(((size_t)rows * cols + kNormElements - 1) / kNormElements); }

struct Front {
    MuonStack grad, momentum;
    bool update, nesterov;
    float mu;
    int rows, cols, parts;
    double* partial;  // [count][parts]
};

__device__ __forceinline__ float direction(float g, float m, bool update, bool nesterov, float mu) {
    return !update ? g : nesterov ? fmaf(mu, m, g) : m;
}

// M <- mu M + G, and the workgroup's share of |U|^2.  In 64 bits: a gradient of 1e-25 or 1e25 has a norm as good as any.
// `V`: four elements at a time, where the arrays are contiguous and allow it; a thread's loads are all under way together.
template <typename GT, int V>
__global__ __launch_bounds__(256) void muon_front_kernel(Front f) {
    constexpr int N = kNormElements / 256 / V;
    const int i = blockIdx.y;
    const GT* const g = static_cast<const GT*>(f.grad.p) + i * f.grad.stride;
    float* const mo = f.update ? static_cast<float*>(const_cast<void*>(f.momentum.p)) + i * f.momentum.stride : nullptr;
    const uint32_t elements = (uint32_t)f.rows * (uint32_t)f.cols, first = blockIdx.x * (uint32_t)kNormElements + threadIdx.x * V;
    float u[N][V], m[N][V];
    uint32_t at[N];
#pragma unroll
    for (int k = 0; k < N; ++k) {
        const uint32_t e = first + k * 256 * V;
        if constexpr (V == 1) {
            const uint32_t r = e / (uint32_t)f.cols, c = e - r * (uint32_t)f.cols;
            at[k] = r * (uint32_t)f.grad.pitch + c;
            u[k][0] = e < elements ? to_f32(g[at[k]]) : 0.0f;
            if (f.update) {
                at[k] = r * (uint32_t)f.momentum.pitch + c;
                m[k][0] = e < elements ? mo[at[k]] : 0.0f;
            }
        } else {
            at[k] = e;
            float4 w = make_float4(0.0f, 0.0f, 0.0f, 0.0f), q = w;
            if (e < elements) {
                if constexpr (sizeof(GT) == 2) {
                    const uint2 h = *reinterpret_cast<const uint2*>(g + e);
                    w = make_float4(__uint_as_float(h.x << 16), __uint_as_float(h.x & 0xffff0000u), __uint_as_float(h.y << 16),
                                    __uint_as_float(h.y & 0xffff0000u));
                } else {
                    w = *reinterpret_cast<const float4*>(g + e);
                }
                if (f.update) q = *reinterpret_cast<const float4*>(mo + e);
            }
            u[k][0] = w.x; u[k][1] = w.y; u[k][2] = w.z; u[k][3] = w.w;
            m[k][0] = q.x; m[k][1] = q.y; m[k][2] = q.z; m[k][3] = q.w;
        }
    }
    double sum = 0.0;
#pragma unroll
    for (int k = 0; k < N; ++k) {
        const bool in = first + k * 256 * V < elements;
        if (f.update) {
#pragma unroll
            for (int v = 0; v < V; ++v) {
                m[k][v] = fmaf(f.mu, m[k][v], u[k][v]);
                u[k][v] = direction(u[k][v], m[k][v], true, f.nesterov, f.mu);
            }
            if (in) {
                if constexpr (V == 4) *reinterpret_cast<float4*>(mo + at[k]) = make_float4(m[k][0], m[k][1], m[k][2], m[k][3]);
                else mo[at[k]] = m[k][0];
            }
        }
#pragma unroll
        for (int v = 0; v < V; ++v) sum += (double)u[k][v] * (double)u[k][v];
    }
    __shared__ double room[4];
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
    if ((threadIdx.x & 63) == 0) room[threadIdx.x >> 6] = sum;
    __syncthreads();
    if (threadIdx.x == 0) f.partial[(size_t)i * f.parts + blockIdx.x] = (room[0] + room[1]) + (room[2] + room[3]);
}

// ---- U into operand order, both ways -------------------------------------------------------------------
// X_k is stored times 2^14 / down, down = 2^-e: e is the largest whole number, 0 at least, for which 1.25 times 2^-e bounds the singular
// values of X_k.  (For an |U|_F of 1.7e-7 and more that is 0 throughout.  At most 98, so that 2^-28 down is a normal number.)
struct Lift {
    float down, up;
};
__device__ __forceinline__ Lift lift_of(double norm, int k) {
    float bound = fminf((float)(norm / (norm + 1e-7)), 1.0f);  // (of a norm that is not a number, too)
    for (int i = 0; i < k; ++i) bound = fminf(bound * 3.4446f, 1.2025f);
    const int e = min(max(ilogbf(1.25f / bound), 0), 98);
    return {ldexpf(1.0f, -e), ldexpf(1.0f, e)};
}

struct Pack {
    Front f;
    Shape s;
    Lift* lift;  // [count][steps]
    int steps;
    bool tall;  // rows > cols: the matrix is taken transposed
    char* x;    // X, X^T of matrix i at i * x_bytes()
    char* xt;
};

// A workgroup takes 32 x 64 of X (m by n).
template <typename GT>
__global__ __launch_bounds__(256) void muon_pack_kernel(Pack a) {
    __shared__ float tile[32][65];
    __shared__ double norm2;
    const Front& f = a.f;
    const int i = blockIdx.z, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const GT* const g = static_cast<const GT*>(f.grad.p) + i * f.grad.stride;
    const float* const mo = f.update ? static_cast<const float*>(f.momentum.p) + i * f.momentum.stride : nullptr;
    const int p0 = blockIdx.x * 32, q0 = blockIdx.y * 64;  // of X
    // element k of this thread: neighbouring threads along the rows as they lie
    auto place = [&](int k, int& p, int& q) {
        p = a.tall ? tid & 31 : k * 4 + wave;
        q = a.tall ? k * 8 + (tid >> 5) : lane;
    };
    float gv[8], m[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        int p, q;
        place(k, p, q);
        const int r = a.tall ? q0 + q : p0 + p, c = a.tall ? p0 + p : q0 + q;
        const bool in = r < f.rows && c < f.cols;
        gv[k] = in ? to_f32(g[(size_t)r * f.grad.pitch + c]) : 0.0f;
        m[k] = in && f.update ? mo[(size_t)r * f.momentum.pitch + c] : 0.0f;
    }
    if (wave == 0) {
        double sum = 0.0;
        for (int p = lane; p < f.parts; p += 64) sum += f.partial[(size_t)i * f.parts + p];
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
        if (lane == 0) norm2 = sum;
    }
    __syncthreads();
    const double norm = sqrt(norm2), factor = (double)kUp * lift_of(norm, 0).up / (norm + 1e-7);
    if (blockIdx.x == 0 && blockIdx.y == 0 && tid < a.steps) a.lift[(size_t)i * a.steps + tid] = lift_of(norm, tid);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        int p, q;
        place(k, p, q);
        tile[p][q] = (float)((double)direction(gv[k], m[k], f.update, f.nesterov, f.mu) * factor);
    }
    __syncthreads();
    // a fragment a wave each way: of X one group of rows and four steps, of X^T two groups and two steps
#pragma unroll
    for (int way = 0; way < 2; ++way) {
        char* const base = (way ? a.xt : a.x) + (size_t)i * a.s.x_bytes();
        const int groups = way ? a.s.ng : a.s.mg, steps = 2 * (way ? a.s.mg : a.s.ng);
        const int group = way ? q0 / 32 + wave / 2 : p0 / 32, step = way ? p0 / 16 + wave % 2 : q0 / 16 + wave;
        if (group >= groups || step >= steps) continue;
        const int row = (way ? 32 * (wave / 2) : 0) + (lane & 31), col = 16 * (way ? wave % 2 : wave) + 8 * (lane >> 5);
        halfx8 hi, lo;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            _Float16 h, l;
            split(way ? tile[col + e][row] : tile[row][col + e], h, l);
            hi[e] = h;
            lo[e] = l;
        }
        char* const at = base + ((size_t)group * steps + step) * kFragment + lane * 16;
        *reinterpret_cast<halfx8*>(at) = hi;
        *reinterpret_cast<halfx8*>(at + 1024) = lo;
    }
}

// ---- products --------------------------------------------------------------------------------------
// C[p][q] = sum_k P[p][k] Q[q][k].
enum Product {
    kGram,   // P = Q = X:        A = C
    kPoly,   // P = Q = A:        B = a I + b A + c C
    kApply,  // P = B, Q = X^T:   X = C, stored both ways
    kLast    // P = B, Q = X^T:   C is the result
};
struct ProductArgs {
    Shape s;
    const char* p;   // operands of matrix 0
    const char* q;
    size_t p_bytes, q_bytes;
    int pg, qg, steps;       // groups of 32 rows of either, steps of 16 of the reduction
    char* direct;            // C^T in operand order: rows q, reduction p
    char* mirrored;          // C in operand order:   rows p, reduction q
    size_t out_bytes;
    const Lift* lift;        // of this step, matrix 0
    int lift_stride;
    // kLast
    MuonStack weight, out;
    bool update, out_bf16, tall;
    bool whole;              // tall, and four neighbouring elements of a row may be accessed at once
    float keep, rate;
};

// What a sum of products is multiplied by.
template <Product kind>
__device__ __forceinline__ float sum_factor(const ProductArgs& a, int matrix) {
    if constexpr (kind == kPoly) return kDown;  // 2^28 C -> 2^14 C
    const Lift* const l = a.lift + (size_t)matrix * a.lift_stride;
    if constexpr (kind == kGram) return kDown * l->down * l->down;
    else if constexpr (kind == kApply) return kDown * l->down * l[1].up;
    else return kDown * kDown * l->down;
}

// byte offset of element (row, column) of an operand with `steps` fragments a group of rows
__device__ __forceinline__ size_t operand_at(int row, int col, int steps) {
    return ((size_t)(row >> 5) * steps + (col >> 4)) * kFragment + ((row & 31) + 32 * ((col >> 3) & 1)) * 16 + (col & 7) * 2;
}

// What a lane reads of 32 x 32 of C's surroundings before it writes its 16 elements: rows 8 j + 4 (lane / 32) .. + 3, j = 0 .. 3, of column
// lane % 32 (those of j at place `at`).
template <Product kind>
struct Before {};
template <>
struct Before<kPoly> {
    halfx4 hi[4], lo[4];  // A
};
template <>
struct Before<kLast> {
    float w[16];
};

__device__ __forceinline__ float* weight_at(const ProductArgs& a, int matrix, int p, int q) {
    return static_cast<float*>(const_cast<void*>(a.weight.p)) + matrix * a.weight.stride +
           (a.tall ? (size_t)q * a.weight.pitch + p : (size_t)p * a.weight.pitch + q);
}

template <Product kind>
__device__ __forceinline__ void read_before(const ProductArgs& a, int matrix, int gp, int gq, int j, int at, int lane, Before<kind>& b) {
    const int p0 = gp * 32 + 8 * j + 4 * (lane >> 5), q = gq * 32 + (lane & 31);
    if constexpr (kind == kPoly) {
        const char* const old = a.q + (size_t)matrix * a.q_bytes + operand_at(q, p0, 2 * a.pg);
        b.hi[at] = *reinterpret_cast<const halfx4*>(old);
        b.lo[at] = *reinterpret_cast<const halfx4*>(old + 1024);
    } else if constexpr (kind == kLast) {
        if (!a.update || q >= a.s.n) return;
        const float* const w = weight_at(a, matrix, p0, q);
        if (a.whole && p0 + 3 < a.s.m) {
            const float4 v = *reinterpret_cast<const float4*>(w);
            b.w[4 * at] = v.x; b.w[4 * at + 1] = v.y; b.w[4 * at + 2] = v.z; b.w[4 * at + 3] = v.w;
        } else {
            const size_t pitch = a.tall ? 1 : a.weight.pitch;
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (p0 + i < a.s.m) b.w[4 * at + i] = w[i * pitch];
        }
    }
}

// Four elements of C, rows p0 .. p0 + 3 (p0 a multiple of 4) of column q, in f32.  `parts`: what was stored of them, hi | lo << 16.
template <Product kind>
__device__ __forceinline__ void write4(const ProductArgs& a, int matrix, int gp, int gq, int j, int at, int lane, const float (&sum)[4],
                                       float factor, const Before<kind>& b, uint32_t (&parts)[4]) {
    const int p0 = gp * 32 + 8 * j + 4 * (lane >> 5), q = gq * 32 + (lane & 31);
    if constexpr (kind == kLast) {
        if (q >= a.s.n) return;
        float o[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] = sum[i] * factor;
        const bool four = a.whole && p0 + 3 < a.s.m;
        if (a.update) {
            float* const w = weight_at(a, matrix, p0, q);
#pragma unroll
            for (int i = 0; i < 4; ++i) o[i] = fmaf(-a.rate, o[i], a.keep * b.w[4 * at + i]);
            if (four) {
                *reinterpret_cast<float4*>(w) = make_float4(o[0], o[1], o[2], o[3]);
            } else {
                const size_t pitch = a.tall ? 1 : a.weight.pitch;
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (p0 + i < a.s.m) w[i * pitch] = o[i];
            }
            return;
        }
        const size_t pitch = a.tall ? 1 : a.out.pitch;
        const size_t e = matrix * a.out.stride + (a.tall ? (size_t)q * a.out.pitch + p0 : (size_t)p0 * a.out.pitch + q);
        if (a.out_bf16) {
            bf16_t* const to = static_cast<bf16_t*>(const_cast<void*>(a.out.p)) + e;
            if (four) {
                *reinterpret_cast<uint2*>(to) = make_uint2(pack2(o[0], o[1]), pack2(o[2], o[3]));
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (p0 + i < a.s.m) to[i * pitch] = from_f32<bf16_t>(o[i]);
            }
        } else {
            float* const to = static_cast<float*>(const_cast<void*>(a.out.p)) + e;
            if (four) {
                *reinterpret_cast<float4*>(to) = make_float4(o[0], o[1], o[2], o[3]);
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (p0 + i < a.s.m) to[i * pitch] = o[i];
            }
        }
    } else {
        halfx4 hi, lo;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float v = sum[i] * factor;
            if constexpr (kind == kPoly) {
                v = fmaf(kB, (float)b.hi[at][i] + (float)b.lo[at][i], kC * v);
                // (the padding's diagonal stays zero)
                if (p0 + i == q && q < a.s.m) v += kA * kUp;
            }
            _Float16 h, l;
            split(v, h, l);
            hi[i] = h;
            lo[i] = l;
            parts[i] = (uint32_t)__builtin_bit_cast(uint16_t, h) | ((uint32_t)__builtin_bit_cast(uint16_t, l) << 16);
        }
        char* const to = a.direct + (size_t)matrix * a.out_bytes + operand_at(q, p0, 2 * a.pg);
        *reinterpret_cast<halfx4*>(to) = hi;
        *reinterpret_cast<halfx4*>(to + 1024) = lo;
    }
}

// Step `half` (columns 16 half .. + 15) of the mirrored fragments of block (gp, gq), from the block's parts as they lie in
// LDS: [column][row], a column every kTurnedPitch words.
constexpr int kTurnedPitch = 36;
__device__ __forceinline__ void write_turned(const ProductArgs& a, int matrix, int gp, int gq, int half, int lane, const uint32_t* turned) {
    uint32_t v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = turned[(16 * half + 8 * (lane >> 5) + e) * kTurnedPitch + (lane & 31)];
    uint4 hi, lo;
    hi.x = __builtin_amdgcn_perm(v[1], v[0], 0x05040100u); hi.y = __builtin_amdgcn_perm(v[3], v[2], 0x05040100u);
    hi.z = __builtin_amdgcn_perm(v[5], v[4], 0x05040100u); hi.w = __builtin_amdgcn_perm(v[7], v[6], 0x05040100u);
    lo.x = __builtin_amdgcn_perm(v[1], v[0], 0x07060302u); lo.y = __builtin_amdgcn_perm(v[3], v[2], 0x07060302u);
    lo.z = __builtin_amdgcn_perm(v[5], v[4], 0x07060302u); lo.w = __builtin_amdgcn_perm(v[7], v[6], 0x07060302u);
    char* const to = a.mirrored + (size_t)matrix * a.out_bytes + ((size_t)gp * 2 * a.qg + 2 * gq + half) * kFragment + lane * 16;
    *reinterpret_cast<uint4*>(to) = hi;
    *reinterpret_cast<uint4*>(to + 1024) = lo;
}

// A and B are symmetric: of a tile's 32 x 32 blocks those above the diagonal are written both ways, those below it not at all.
template <Product kind>
constexpr bool kSymmetric = kind == kGram || kind == kPoly;

// ---- few tiles: the reduction split over a workgroup's waves ----------------------------------------------
// Tile t of the upper triangle (with the diagonal), counted by columns: (row, column) with row <= column.
__device__ __forceinline__ void triangle(int t, int& row, int& col) {
    int c = (int)((sqrtf(8.0f * (float)t + 1.0f) - 1.0f) * 0.5f);
    while ((c + 1) * (c + 2) / 2 <= t) ++c;
    while (c * (c + 1) / 2 > t) --c;
    col = c;
    row = t - c * (c + 1) / 2;
}

// A workgroup takes B x B blocks of 32 x 32 of C, and each of its W waves every W-th piece of the reduction, straight from the caches to
// its registers: nothing to wait for but the loads themselves, most of which are under way at once.  The waves' sums meet in LDS.
template <Product kind, int B, int W>
__global__ __launch_bounds__(64 * W) void muon_product_split_kernel(ProductArgs a) {
    constexpr int S = B == 1 ? 4 : 2;        // steps of a piece
    constexpr int kQuads = B * B * 4;        // (block, j): four elements a lane
    __shared__ __align__(16) float4 room[W * kQuads * 64];
    static_assert(sizeof(room) >= B * B * 32 * kTurnedPitch * 4, "the turned blocks take the sums' place");
    const int matrix = blockIdx.y, lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int tp, tq;
    if constexpr (kSymmetric<kind>) {
        triangle(blockIdx.x, tp, tq);
    } else {
        const int rows = (a.pg + B - 1) / B;
        tp = blockIdx.x % rows;
        tq = blockIdx.x / rows;
    }
    const char* const pm = a.p + (size_t)matrix * a.p_bytes;
    const char* const qm = a.q + (size_t)matrix * a.q_bytes;
    const float factor = sum_factor<kind>(a, matrix);
    const __amdgpu_buffer_rsrc_t p_buffer = __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(pm), 0, (int)a.p_bytes, kRawBuffer);
    const __amdgpu_buffer_rsrc_t q_buffer = __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(qm), 0, (int)a.q_bytes, kRawBuffer);
    int ps[B], qs[B];
#pragma unroll
    for (int i = 0; i < B; ++i) {
        ps[i] = min(tp * B + i, a.pg - 1) * a.steps * kFragment;
        qs[i] = min(tq * B + i, a.qg - 1) * a.steps * kFragment;
    }
    struct Piece {
        halfx8 ph[S][B], pl[S][B], qh[S][B], ql[S][B];
    };
    const int at = lane * 16;
    auto load = [&](Piece& d, int piece) {
#pragma unroll
        for (int k = 0; k < S; ++k) {
            const int step = min(piece * S + k, a.steps - 1) * kFragment;
#pragma unroll
            for (int i = 0; i < B; ++i) {
                d.ph[k][i] = __builtin_bit_cast(halfx8, __builtin_amdgcn_raw_buffer_load_b128(p_buffer, at, ps[i] + step, kVolatile));
                d.pl[k][i] = __builtin_bit_cast(halfx8, __builtin_amdgcn_raw_buffer_load_b128(p_buffer, at + 1024, ps[i] + step, kVolatile));
                d.qh[k][i] = __builtin_bit_cast(halfx8, __builtin_amdgcn_raw_buffer_load_b128(q_buffer, at, qs[i] + step, kVolatile));
                d.ql[k][i] = __builtin_bit_cast(halfx8, __builtin_amdgcn_raw_buffer_load_b128(q_buffer, at + 1024, qs[i] + step, kVolatile));
            }
        }
    };
    floatx16 acc[B][B];
#pragma unroll
    for (int r = 0; r < B; ++r)
#pragma unroll
        for (int c = 0; c < B; ++c) acc[r][c] = floatx16{};
    auto multiply = [&](const Piece& d, int piece) {
#pragma unroll
        for (int k = 0; k < S; ++k) {
            if (piece * S + k >= a.steps) break;
#pragma unroll
            for (int part = 0; part < 3; ++part)
#pragma unroll
                for (int r = 0; r < B; ++r)
#pragma unroll
                    for (int c = 0; c < B; ++c)
                        acc[r][c] = __builtin_amdgcn_mfma_f32_32x32x16_f16(part == 0 ? d.pl[k][r] : d.ph[k][r],
                                                                           part == 1 ? d.ql[k][c] : d.qh[k][c], acc[r][c], 0, 0, 0);
        }
    };
    const int pieces = (a.steps + S - 1) / S;
    Piece one, two;
    if (wave < pieces) load(one, wave);
    for (int piece = wave; piece < pieces; piece += 2 * W) {
        if (piece + W < pieces) load(two, piece + W);
        __builtin_amdgcn_sched_barrier(0);
        multiply(one, piece);
        if (piece + W >= pieces) break;
        if (piece + 2 * W < pieces) load(one, piece + 2 * W);
        __builtin_amdgcn_sched_barrier(0);
        multiply(two, piece + W);
    }
#pragma unroll
    for (int r = 0; r < B; ++r)
#pragma unroll
        for (int c = 0; c < B; ++c)
#pragma unroll
            for (int j = 0; j < 4; ++j)
                room[(wave * kQuads + (r * B + c) * 4 + j) * 64 + lane] =
                    make_float4(acc[r][c][4 * j], acc[r][c][4 * j + 1], acc[r][c][4 * j + 2], acc[r][c][4 * j + 3]);
    // a wave adds and writes every W-th quad
    constexpr int T = (kQuads + W - 1) / W;
    auto block_of = [&](int t, int& gp, int& gq, int& j) {  // false: nothing to write there
        const int quad = wave + t * W;
        j = quad % 4;
        gp = tp * B + quad / 4 / B;
        gq = tq * B + quad / 4 % B;
        return quad < kQuads && gp < a.pg && gq < a.qg && !(kSymmetric<kind> && gp > gq);
    };
    Before<kind> before[T];
#pragma unroll
    for (int t = 0; t < T; ++t) {
        int gp, gq, j;
        if (block_of(t, gp, gq, j)) read_before<kind>(a, matrix, gp, gq, j, 0, lane, before[t]);
    }
    __syncthreads();
    float sum[T][4];
#pragma unroll
    for (int t = 0; t < T; ++t) {
        const int quad = min(wave + t * W, kQuads - 1);
        float4 v = room[quad * 64 + lane];
#pragma unroll
        for (int w = 1; w < W; ++w) {
            const float4 x = room[(w * kQuads + quad) * 64 + lane];
            v.x += x.x; v.y += x.y; v.z += x.z; v.w += x.w;
        }
        sum[t][0] = v.x; sum[t][1] = v.y; sum[t][2] = v.z; sum[t][3] = v.w;
    }
    __syncthreads();  // the sums have been read: the turned blocks, for the mirrored operand, take their place
    uint32_t* const turned = reinterpret_cast<uint32_t*>(room);
#pragma unroll
    for (int t = 0; t < T; ++t) {
        int gp, gq, j;
        if (!block_of(t, gp, gq, j)) continue;
        uint32_t parts[4];
        write4<kind>(a, matrix, gp, gq, j, 0, lane, sum[t], factor, before[t], parts);
        if constexpr (kind != kLast)
            *reinterpret_cast<uint4*>(turned + (((wave + t * W) / 4) * 32 + (lane & 31)) * kTurnedPitch + 8 * j + 4 * (lane >> 5)) =
                make_uint4(parts[0], parts[1], parts[2], parts[3]);
    }
    if constexpr (kind != kLast) {
        __syncthreads();
        for (int i = wave; i < B * B * 2; i += W) {
            const int block = i / 2, gp = tp * B + block / B, gq = tq * B + block % B;
            if (gp < a.pg && gq < a.qg && !(kSymmetric<kind> && gp >= gq))
                write_turned(a, matrix, gp, gq, i % 2, lane, turned + block * 32 * kTurnedPitch);
        }
    }
}

// f(integral_constant<int, I>) ... f(integral_constant<int, N - 1>), in order
template <int I, int N, typename F>
__device__ __forceinline__ void for_each_block(F&& f) {
    if constexpr (I < N) {
        f(std::integral_constant<int, I>{});
        for_each_block<I + 1, N>(f);
    }
}

// ---- many tiles ------------------------------------------------------------------------------------
// A workgroup takes 32 RG rows (p) by 128 CG columns (q) of C, four waves side by side along the columns.  The rows'
// operand goes through LDS, 32 of the reduction (a chunk) at a time in two stages, and is read by all four waves; the columns'
// operand is a wave's own and goes to its registers, two steps of 16 ahead.
//
// A step's multiplies go unit by unit, a unit being two accumulators (so that a multiply never waits for the one in front of
// it); a unit's row fragments are taken from LDS as soon as the unit in front of them in time is done with the registers (CG = 2), or
// a whole step ahead (CG = 1, where registers are plenty).  Stage s of a chunk is read for the last time in the chunk's first step, and
// the barrier of the chunk stands behind the first unit of its second step: behind it the next chunk's stage is complete and this
// one's free.  Loads go out a chunk (rows) and two steps (columns) ahead.  Scheduling barriers keep all of that in place: left to
// itself the compiler moves every load down to its use, which takes 2.2 times as long.
template <Product kind, int RG, int CG>
__global__ __launch_bounds__(256, 2) void muon_product_kernel(ProductArgs a, int tiles, int total) {
    constexpr int kStage = RG * 4096;  // bytes
    constexpr int U = RG * CG / 2, FB = CG == 2 ? 1 : 2;    // units, sets of row fragments
    constexpr int PD = CG == 2 ? 1 : 3, QD = CG == 2 ? 3 : 6;  // chunks of rows, steps of columns in registers
    static_assert(6 % QD == 0 && 3 % PD == 0, "three chunks are written out");
    __shared__ __align__(16) char lds[2 * kStage > 4 * 32 * kTurnedPitch * 4 ? 2 * kStage : 4 * 32 * kTurnedPitch * 4];
    // neighbouring tiles on one XCD, whose second-level cache then holds the operands that they share
    const int share = (total + 7) / 8, w = (int)(blockIdx.x % 8) * share + (int)(blockIdx.x / 8);
    if ((int)(blockIdx.x / 8) >= share || w >= total) return;
    const int matrix = w / tiles;
    int tile = w - matrix * tiles, tp, tq;
    const int rows = (a.pg + RG - 1) / RG;
    // (on the diagonal a wave's work grows with its column: which of the compute unit's four SIMDs gets how much goes round)
    const int turn = tile;
    if constexpr (kSymmetric<kind>) {
        for (tq = 0;; ++tq) {
            const int n = (min((tq + 1) * 4 * CG, a.qg) - 1) / RG + 1;  // row tiles that reach above the diagonal
            if (tile < n) break;
            tile -= n;
        }
        tp = tile;
    } else {
        tp = tile % rows;
        tq = tile / rows;
    }
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int chunks = a.steps / 2;
    const char* const pm = a.p + (size_t)matrix * a.p_bytes;
    const char* const qm = a.q + (size_t)matrix * a.q_bytes;
    const int p0 = tp * RG, q0 = tq * 4 * CG + ((wave + turn) & 3) * CG;  // groups
    // row groups that the wave has something to do for: inside C, and above the diagonal for one of its columns
    const int live = q0 >= a.qg ? 0 : min(a.pg - p0, kSymmetric<kind> ? q0 + CG - p0 : RG);
    // Loads through a buffer descriptor: its base and the part of the offset that goes up with the reduction are scalars, so the loop
    // holds one vector register of addresses.  (An operand of one matrix has at most 2^30 bytes.)  A thread's pieces of a stage: piece i
    // of group i, whose two steps of 16 lie side by side.
    const float factor = sum_factor<kind>(a, matrix);
    const __amdgpu_buffer_rsrc_t p_buffer = __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(pm), 0, (int)a.p_bytes, kRawBuffer);
    const __amdgpu_buffer_rsrc_t q_buffer = __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(qm), 0, (int)a.q_bytes, kRawBuffer);
    const int p_at = tid * 16, q_at = lane * 16;
    int ps[RG], qs[CG];
#pragma unroll
    for (int i = 0; i < RG; ++i) ps[i] = min(p0 + i, a.pg - 1) * a.steps * kFragment;
#pragma unroll
    for (int c = 0; c < CG; ++c) qs[c] = min(q0 + c, a.qg - 1) * a.steps * kFragment;

    // (loads that stay where they are written: the compiler moves others behind a branch, next to their use)
    u32x4 next[PD][RG];
    halfx8 qh[QD][CG], ql[QD][CG], ph[FB][RG], pl[FB][RG];
    auto load_p = [&](int set, int chunk) {
        const int k = min(chunk, chunks - 1);
#pragma unroll
        for (int i = 0; i < RG; ++i) next[set][i] = __builtin_amdgcn_raw_buffer_load_b128(p_buffer, p_at, ps[i] + k * 2 * kFragment, kVolatile);
    };
    auto store_p = [&](int set, int chunk) {
#pragma unroll
        for (int i = 0; i < RG; ++i) *reinterpret_cast<u32x4*>(lds + (chunk & 1) * kStage + i * 4096 + tid * 16) = next[set][i];
    };
    auto load_q = [&](int slot, int step) {
        const int k = min(step, a.steps - 1);
#pragma unroll
        for (int c = 0; c < CG; ++c) {
            qh[slot][c] = __builtin_bit_cast(halfx8, __builtin_amdgcn_raw_buffer_load_b128(q_buffer, q_at, qs[c] + k * kFragment, kVolatile));
            ql[slot][c] = __builtin_bit_cast(halfx8, __builtin_amdgcn_raw_buffer_load_b128(q_buffer, q_at + 1024, qs[c] + k * kFragment, kVolatile));
        }
    };
    auto take_p = [&](int set, int chunk, int half, int unit) {  // the unit's row fragments
        const unsigned char* const at = reinterpret_cast<unsigned char*>(lds) + (chunk & 1) * kStage + half * kFragment + lane * 16;
#pragma unroll
        for (int r = unit * RG / U; r < (unit + 1) * RG / U; ++r) {
            ph[set][r] = lds_load_ahead<halfx8>(at + r * 4096);
            pl[set][r] = lds_load_ahead<halfx8>(at + r * 4096 + 1024);
        }
    };
    floatx16 acc[RG][CG];
#pragma unroll
    for (int r = 0; r < RG; ++r)
#pragma unroll
        for (int c = 0; c < CG; ++c) acc[r][c] = floatx16{};

    // (in the order in which the loop issues them: its waits count the loads that are younger)
    load_p(0, 0);
    load_q(0, 0);
    store_p(0, 0);
    if constexpr (PD == 1) {
        load_p(0, 1);
        load_q(1, 1);
    } else {
#pragma unroll
        for (int i = 1; i < PD; ++i) {
            load_p(i, i);
            load_q(2 * i - 1, 2 * i - 1);
            load_q(2 * i, 2 * i);
        }
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < U; ++u) take_p(0, 0, 0, u);
    // one chunk; `number`: its number modulo 3, which says where what it reads lies
    auto multiply = [&](auto number, int chunk) {
        constexpr int n = decltype(number)::value;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const int slot = (2 * n + half) % QD, set = FB == 1 ? 0 : half;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                // memory instructions of the unit: in front of its multiplies where fragments have a set of their own
                auto memory = [&] {
                    __builtin_amdgcn_sched_barrier(0);
                    if (u == 0) {
                        if (half == 0) {
                            store_p((n + 1) % PD, chunk + 1);
                            load_p(PD == 1 ? 0 : n % PD, chunk + (PD == 1 ? 2 : PD));
                        } else {
                            __syncthreads();
                        }
                        load_q((slot + QD - 1) % QD, 2 * chunk + half + QD - 1);
                    }
                    take_p(FB == 1 ? 0 : 1 - half, chunk + half, 1 - half, u);
                    __builtin_amdgcn_sched_barrier(0);
                };
                if constexpr (FB == 2) memory();
                if (u * RG / U < live) {
#pragma unroll
                    for (int part = 0; part < 3; ++part)
#pragma unroll
                        for (int r = u * RG / U; r < (u + 1) * RG / U; ++r)
#pragma unroll
                            for (int c = 0; c < CG; ++c)
                                acc[r][c] = __builtin_amdgcn_mfma_f32_32x32x16_f16(
                                    part == 0 ? pl[set][r] : ph[set][r], part == 1 ? ql[slot][c] : qh[slot][c], acc[r][c], 0, 0, 0);
                }
                if constexpr (FB == 1) memory();
            }
        }
    };
    int chunk = 0;
    for (; chunk + 3 <= chunks; chunk += 3) {
        multiply(std::integral_constant<int, 0>{}, chunk);
        multiply(std::integral_constant<int, 1>{}, chunk + 1);
        multiply(std::integral_constant<int, 2>{}, chunk + 2);
    }
    if (chunk < chunks) multiply(std::integral_constant<int, 0>{}, chunk);
    if (chunk + 1 < chunks) multiply(std::integral_constant<int, 1>{}, chunk + 1);
    __syncthreads();
    // (the stages are free)
    uint32_t* const turned = reinterpret_cast<uint32_t*>(lds) + wave * 32 * kTurnedPitch;
    auto wanted = [&](int gp, int gq) { return gp < a.pg && gq < a.qg && !(kSymmetric<kind> && gp > gq); };
    // (what a block reads is asked for before the block in front of it is written)
    Before<kind> before[2];
    auto ask = [&](auto block) {
        constexpr int b = decltype(block)::value;
        if (wanted(p0 + b / CG, q0 + b % CG))
#pragma unroll
            for (int j = 0; j < 4; ++j) read_before<kind>(a, matrix, p0 + b / CG, q0 + b % CG, j, j, lane, before[b % 2]);
    };
    ask(std::integral_constant<int, 0>{});
    for_each_block<0, RG * CG>([&](auto block) {
        constexpr int b = decltype(block)::value, r = b / CG, c = b % CG;
        if constexpr (b + 1 < RG * CG) ask(std::integral_constant<int, b + 1>{});
        const int gp = p0 + r, gq = q0 + c;
        if (!wanted(gp, gq)) return;
        const bool mirror = kind == kApply || (kSymmetric<kind> && gp != gq);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float sum[4] = {acc[r][c][4 * j], acc[r][c][4 * j + 1], acc[r][c][4 * j + 2], acc[r][c][4 * j + 3]};
            uint32_t parts[4];
            write4<kind>(a, matrix, gp, gq, j, j, lane, sum, factor, before[b % 2], parts);
            if (mirror)
                *reinterpret_cast<uint4*>(turned + (lane & 31) * kTurnedPitch + 8 * j + 4 * (lane >> 5)) =
                    make_uint4(parts[0], parts[1], parts[2], parts[3]);
        }
        if (mirror) {
            // (the wave's own room: its LDS instructions are carried out in order)
            __builtin_amdgcn_wave_barrier();
            write_turned(a, matrix, gp, gq, 0, lane, turned);
            write_turned(a, matrix, gp, gq, 1, lane, turned);
            __builtin_amdgcn_wave_barrier();
        }
    });
}

constexpr int kUnits = 256;  // compute units

template <Product kind, int RG, int CG>
int tiles_of(const ProductArgs& a) {
    const int rows = (a.pg + RG - 1) / RG, cols = (a.qg + 4 * CG - 1) / (4 * CG);
    if (!kSymmetric<kind>) return rows * cols;
    int n = 0;
    for (int q = 0; q < cols; ++q) n += (std::min((q + 1) * 4 * CG, a.qg) - 1) / RG + 1;
    return n;
}

template <Product kind, int RG, int CG>
hipError_t launch_tiles(const ProductArgs& a, int count, hipStream_t s) {
    const int tiles = tiles_of<kind, RG, CG>(a), total = tiles * count;
    hipLaunchKernelGGL((muon_product_kernel<kind, RG, CG>), dim3((total + 7) / 8 * 8), dim3(256), 0, s, a, tiles, total);
    return hipGetLastError();
}

template <Product kind, int B>
int split_tiles_of(const ProductArgs& a) {
    const int rows = (a.pg + B - 1) / B, cols = (a.qg + B - 1) / B;
    return kSymmetric<kind> ? rows * (rows + 1) / 2 : rows * cols;
}

template <Product kind, int B, int W>
hipError_t launch_split(const ProductArgs& a, int count, hipStream_t s) {
    hipLaunchKernelGGL((muon_product_split_kernel<kind, B, W>), dim3(split_tiles_of<kind, B>(a), count), dim3(64 * W), 0, s, a);
    return hipGetLastError();
}

// Which kernel takes a product.  us a call of five steps (17 launches), count x [rows, cols], by 32 x 32 split eightfold / 64 x 64 split
// fourfold / 64 x 128 / 128 x 256:
//   1 x [512, 512] 84 / 125 / 158 / 383, 1 x [768, 768] 141 / 141 / 208 / 515, 1 x [1024, 1024] 228 / 180 / 239 / 635, 1 x [1408, 1408] 487 / 294 / 334 /
//   813, 4 x [352, 512] 125 / 122 / 142 / 331, 8 x [352, 512] 195 / 156 / 145 / 337, 16 x [352, 512] 319 / 254 / 186 / 349, 24 x [227, 341] 240 / 172 /
//   148 / 292, 4 x [768, 1408] 526 / 427 / 351 / 624, 128 x [64, 64] 91 / 72 / 82 / 104.
// What tells them apart is how many workgroups a launch has: under two 64 x 64 tiles for every five compute units the reduction
// has to be split to use them, and from four for every five on the larger tiles' smaller traffic counts.  128 x 256 (twice the
// multiplies for every byte) needs two workgroups a unit: 16 x [768, 1408], 192 of them for A 62 us / 72, 576 for X 117 / 106; 128 x [704, 1024], 1536
// for A 305 / 272, for X twice as many 553 / 430.
template <Product kind>
MuonTile tile_of(const ProductArgs& a, int count) {
    const long long tiles = (long long)split_tiles_of<kind, 2>(a) * count;  // of 64 x 64
    if (tiles * 5 <= kUnits * 2) return MuonTile::Split32;
    if (tiles * 5 <= kUnits * 4) return MuonTile::Split64;
    return (long long)tiles_of<kind, 4, 2>(a) * count < 2 * kUnits ? MuonTile::Rows64 : MuonTile::Rows128;
}

template <Product kind>
hipError_t launch_product(const ProductArgs& a, int count, hipStream_t s) {
    switch (tile_of<kind>(a, count)) {
        case MuonTile::Split32: return launch_split<kind, 1, 8>(a, count, s);
        case MuonTile::Split64: return launch_split<kind, 2, 4>(a, count, s);
        case MuonTile::Rows64: return launch_tiles<kind, 2, 1>(a, count, s);
        case MuonTile::Rows128: break;
    }
    return launch_tiles<kind, 4, 2>(a, count, s);
}

size_t rounded(size_t bytes) { return (bytes + 255) & ~(size_t)255; }

}  // namespace

MuonTile muon_tile(int count, int rows, int cols, int product) {
    const Shape s = shape_of(rows, cols);
    ProductArgs a{};
    a.s = s;
    a.pg = s.mg;
    a.qg = product == 2 ? s.ng : s.mg;
    return product == 2 ? tile_of<kApply>(a, count) : tile_of<kGram>(a, count);
}

size_t muon_workspace_bytes(int count, int rows, int cols) {
    const Shape s = shape_of(rows, cols);
    return rounded((size_t)count * norm_parts(rows, cols) * 8) + rounded((size_t)count * kMostMuonSteps * sizeof(Lift)) +
           count * (3 * s.x_bytes() + 2 * s.a_bytes());
}

hipError_t launch_muon(const MuonCall& c, hipStream_t s) {
    const Shape sh = shape_of(c.rows, c.cols);
    const bool update = c.weight.p != nullptr, tall = c.rows > c.cols;
    Front f{c.grad, c.momentum, update, c.nesterov, c.mu, c.rows, c.cols, norm_parts(c.rows, c.cols),
            static_cast<double*>(c.workspace)};
    char* at = static_cast<char*>(c.workspace) + rounded((size_t)c.count * f.parts * 8);
    Lift* const lift = reinterpret_cast<Lift*>(at);
    at += rounded((size_t)c.count * kMostMuonSteps * sizeof(Lift));
    char *x, *xt[2], *am, *bm;
    x = at;  // (a step that writes X reads X^T alone, which lies in two places in turn)
    at += c.count * sh.x_bytes();
    for (char*& p : xt) {
        p = at;
        at += c.count * sh.x_bytes();
    }
    am = at;
    bm = at + c.count * sh.a_bytes();
    const dim3 fg(f.parts, c.count), pgrid(sh.mg, (sh.ng + 1) / 2, c.count);
    const Pack pk{f, sh, lift, c.steps, tall, x, xt[0]};
    const size_t elements = (size_t)c.rows * c.cols;
    auto fours = [&](const MuonStack& st, int size) {  // four neighbouring elements at once, wherever they stand
        return st.pitch == c.cols && elements % 4 == 0 && (c.count == 1 || st.stride % 4 == 0) && reinterpret_cast<uintptr_t>(st.p) % (4 * size) == 0;
    };
    const bool four = fours(c.grad, c.grad_bf16 ? 2 : 4) && (!update || fours(c.momentum, 4));
    if (c.grad_bf16) {
        if (four) hipLaunchKernelGGL((muon_front_kernel<bf16_t, 4>), fg, dim3(256), 0, s, f);
        else hipLaunchKernelGGL((muon_front_kernel<bf16_t, 1>), fg, dim3(256), 0, s, f);
        hipLaunchKernelGGL(muon_pack_kernel<bf16_t>, pgrid, dim3(256), 0, s, pk);
    } else {
        if (four) hipLaunchKernelGGL((muon_front_kernel<float, 4>), fg, dim3(256), 0, s, f);
        else hipLaunchKernelGGL((muon_front_kernel<float, 1>), fg, dim3(256), 0, s, f);
        hipLaunchKernelGGL(muon_pack_kernel<float>, pgrid, dim3(256), 0, s, pk);
    }
    hipError_t e = hipGetLastError();
    for (int k = 0; k < c.steps && e == hipSuccess; ++k) {
        const int now = k & 1;
        ProductArgs g{};
        g.s = sh;
        g.p = g.q = x;
        g.p_bytes = g.q_bytes = sh.x_bytes();
        g.pg = g.qg = sh.mg;
        g.steps = 2 * sh.ng;
        g.lift = lift + k;
        g.lift_stride = c.steps;
        g.direct = g.mirrored = am;
        g.out_bytes = sh.a_bytes();
        e = launch_product<kGram>(g, c.count, s);
        if (e != hipSuccess) break;
        g.p = g.q = am;
        g.p_bytes = g.q_bytes = sh.a_bytes();
        g.steps = 2 * sh.mg;
        g.direct = g.mirrored = bm;
        e = launch_product<kPoly>(g, c.count, s);
        if (e != hipSuccess) break;
        g.p = bm;
        g.q = xt[now];
        g.q_bytes = g.out_bytes = sh.x_bytes();
        g.qg = sh.ng;
        g.direct = xt[1 - now];
        g.mirrored = x;
        if (k + 1 < c.steps) {
            e = launch_product<kApply>(g, c.count, s);
        } else {
            g.weight = c.weight;
            g.out = c.out;
            g.update = update;
            g.out_bf16 = c.out_bf16;
            g.tall = tall;
            const MuonStack& to = update ? c.weight : c.out;
            const bool half = !update && c.out_bf16;
            g.whole = tall && to.pitch % 4 == 0 && to.stride % 4 == 0 && reinterpret_cast<uintptr_t>(to.p) % (half ? 8 : 16) == 0;
            g.keep = c.keep;
            g.rate = c.rate;
            e = launch_product<kLast>(g, c.count, s);
        }
    }
    return e;
}

}  // namespace rbmoe
