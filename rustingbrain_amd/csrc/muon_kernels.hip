// Orthogonalised updates: the quintic Newton-Schulz iteration on the matrix cores, and the optimiser step around it.
//
//   X0 = U / (|U|_F + 1e-7)                                  [m, n] with m <= n: a taller matrix is taken transposed
//   A = X X^T,  B = b A + c A A,  X <- a X + B X             (a, b, c) = (3.4445, -4.7750, 2.0315), `steps` times
//
// acts on the singular values alone, p(s) = a s + b s^3 + c s^5: p maps [0, 1.2025] into itself, and five steps bring everything from
// 0.003 up into [0.68, 1.21].  So throughout |X| <= 1.21, |A| <= 1.47 and |B| <= 2.81 (spectral norms, which bound the elements).
//
// Precision.  The result is f32-grade: every operand is kept as two fp16 numbers, hi = fp16(2^14 v) and lo = fp16(2^14 v - hi), together 22
// bits; the bounds above keep 2^14 v below 65504, and an element as small as 2^-26 still has its bits.  A product is three on the matrix
// cores, hi hi + hi lo + lo hi, with f32 sums; what is left out is 2^-22 of a term.  That is three fp16 products at 16 times the rate of
// the f32 ones.  (Two bf16 parts hold 16 bits, and five steps of them end 1e-5 from the exact result where f32 ends 2e-6.)
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

typedef __attribute__((__vector_size__(8 * sizeof(_Float16)))) _Float16 halfx8;
typedef __attribute__((__vector_size__(4 * sizeof(_Float16)))) _Float16 halfx4;

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
constexpr int kNormElements = 8192;  // of one workgroup
int norm_parts(int rows, int cols) { return (int)(((size_t)rows * cols + kNormElements - 1) / kNormElements); }

struct Front {
    MuonStack grad, momentum;
    bool update, nesterov;
    float mu;
    int rows, cols, parts;
    double* partial;  // [count][parts]
};

template <typename GT>
__device__ __forceinline__ float direction(float g, float m, bool update, bool nesterov, float mu) {
    return !update ? g : nesterov ? fmaf(mu, m, g) : m;
}

// M <- mu M + G, and the workgroup's share of |U|^2.  In 64 bits: a gradient of 1e-25 or 1e25 has a norm as good as any.
template <typename GT>
__global__ __launch_bounds__(256) void muon_front_kernel(Front f) {
    const int i = blockIdx.y;
    const GT* const g = static_cast<const GT*>(f.grad.p) + i * f.grad.stride;
    float* const mo = f.update ? static_cast<float*>(const_cast<void*>(f.momentum.p)) + i * f.momentum.stride : nullptr;
    const size_t elements = (size_t)f.rows * f.cols, first = (size_t)blockIdx.x * kNormElements;
    double sum = 0.0;
    for (int k = 0; k < kNormElements / 256; ++k) {
        const size_t e = first + (size_t)k * 256 + threadIdx.x;
        if (e >= elements) break;
        const int r = (int)(e / (unsigned)f.cols), c = (int)(e - (size_t)r * f.cols);
        const float gv = to_f32(g[(size_t)r * f.grad.pitch + c]);
        float u = gv;
        if (f.update) {
            float* const p = mo + (size_t)r * f.momentum.pitch + c;
            const float m = fmaf(f.mu, *p, gv);
            *p = m;
            u = direction<GT>(gv, m, true, f.nesterov, f.mu);
        }
        sum += (double)u * (double)u;
    }
    __shared__ double room[4];
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
    if ((threadIdx.x & 63) == 0) room[threadIdx.x >> 6] = sum;
    __syncthreads();
    if (threadIdx.x == 0) f.partial[(size_t)i * f.parts + blockIdx.x] = (room[0] + room[1]) + (room[2] + room[3]);
}

// ---- U into operand order, both ways -------------------------------------------------------------------
struct Pack {
    Front f;
    Shape s;
    bool tall;  // rows > cols: the matrix is taken transposed
    char* x;    // X, X^T of matrix i at i * x_bytes()
    char* xt;
};

// A workgroup takes 64 x 64 of X (m by n).
template <typename GT>
__global__ __launch_bounds__(256) void muon_pack_kernel(Pack a) {
    __shared__ float tile[64][65];
    __shared__ double norm2;
    const Front& f = a.f;
    const int i = blockIdx.z, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    if (wave == 0) {
        double sum = 0.0;
        for (int p = lane; p < f.parts; p += 64) sum += f.partial[(size_t)i * f.parts + p];
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
        if (lane == 0) norm2 = sum;
    }
    __syncthreads();
    const double factor = (double)kUp / (sqrt(norm2) + 1e-7);
    const GT* const g = static_cast<const GT*>(f.grad.p) + i * f.grad.stride;
    const float* const mo = f.update ? static_cast<const float*>(f.momentum.p) + i * f.momentum.stride : nullptr;
    const int p0 = blockIdx.x * 64, q0 = blockIdx.y * 64;  // of X
    const int r0 = a.tall ? q0 : p0, c0 = a.tall ? p0 : q0; // of the matrix as it lies
#pragma unroll
    for (int k = 0; k < 16; ++k) {
        const int r = r0 + k * 4 + wave, c = c0 + lane;
        float v = 0.0f;
        if (r < f.rows && c < f.cols) {
            const float gv = to_f32(g[(size_t)r * f.grad.pitch + c]);
            const float m = f.update ? mo[(size_t)r * f.momentum.pitch + c] : 0.0f;
            v = (float)((double)direction<GT>(gv, m, f.update, f.nesterov, f.mu) * factor);
        }
        if (a.tall) tile[lane][k * 4 + wave] = v; else tile[k * 4 + wave][lane] = v;
    }
    __syncthreads();
    // 2 groups of rows x 4 columns steps x 64 lanes, each way
#pragma unroll
    for (int way = 0; way < 2; ++way) {
        char* const base = (way ? a.xt : a.x) + (size_t)i * a.s.x_bytes();
        const int groups = way ? a.s.ng : a.s.mg, steps = 2 * (way ? a.s.mg : a.s.ng);
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const int block = k * 4 + wave;
            const int group = (way ? q0 : p0) / 32 + block / 4, step = (way ? p0 : q0) / 16 + block % 4;
            if (group >= groups || step >= steps) continue;
            const int row = (block / 4) * 32 + (lane & 31), col = (block % 4) * 16 + 8 * (lane >> 5);
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
}

// ---- products --------------------------------------------------------------------------------------
// C[p][q] = sum_k P[p][k] Q[q][k].
enum Product {
    kGram,   // P = Q = X:        A = C, stored
    kPoly,   // P = Q = A:        B = b A + c C, stored
    kApply,  // P = B, Q = X^T:   X = a X + C, stored both ways
    kLast    // P = B, Q = X^T:   a X + C is the result
};
struct ProductArgs {
    Shape s;
    const char* p;   // operands of matrix 0
    const char* q;
    size_t p_bytes, q_bytes;
    int pg, qg, steps;       // groups of 32 rows of either, steps of 16 of the reduction
    const char* old;         // kPoly: A; kApply, kLast: X^T (the operand whose rows are C's columns)
    char* direct;            // C^T in operand order: rows q, reduction p
    char* mirrored;          // C in operand order:   rows p, reduction q
    size_t out_bytes;
    // kLast
    MuonStack weight, out;
    bool update, out_bf16, tall;
    float keep, rate;
};

// byte offset of element (row, column) of an operand with `steps` fragments a group of rows
__device__ __forceinline__ size_t operand_at(int row, int col, int steps) {
    return ((size_t)(row >> 5) * steps + (col >> 4)) * kFragment + ((row & 31) + 32 * ((col >> 3) & 1)) * 16 + (col & 7) * 2;
}

// Four elements of C, rows p0 .. p0 + 3 (p0 a multiple of 4) of column q, in f32.
template <Product kind>
__device__ __forceinline__ void write4(const ProductArgs& a, int matrix, int p0, int q, bool mirror, const float (&sum)[4]) {
    float v[4];
    const size_t at = operand_at(q, p0, 2 * a.pg);  // (the four lie side by side)
    if constexpr (kind == kGram) {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = sum[i] * kDown;  // 2^28 A -> 2^14 A
    } else {
        const char* const old = a.old + (size_t)matrix * a.out_bytes + at;
        const halfx4 hi = *reinterpret_cast<const halfx4*>(old), lo = *reinterpret_cast<const halfx4*>(old + 1024);
        constexpr float own = kind == kPoly ? kB : kA, other = kind == kPoly ? kC : 1.0f;
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = fmaf(own, (float)hi[i] + (float)lo[i], other * kDown * sum[i]);
    }
    if constexpr (kind == kLast) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int p = p0 + i;
            if (p >= a.s.m || q >= a.s.n) continue;
            const int r = a.tall ? q : p, c = a.tall ? p : q;
            const float o = v[i] * kDown;
            if (a.update) {
                float* const w = static_cast<float*>(const_cast<void*>(a.weight.p)) + matrix * a.weight.stride + (size_t)r * a.weight.pitch + c;
                *w = fmaf(-a.rate, o, a.keep * *w);
            } else {
                const size_t e = matrix * a.out.stride + (size_t)r * a.out.pitch + c;
                if (a.out_bf16) static_cast<bf16_t*>(const_cast<void*>(a.out.p))[e] = from_f32<bf16_t>(o);
                else static_cast<float*>(const_cast<void*>(a.out.p))[e] = o;
            }
        }
    } else {
        halfx4 hi, lo;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            _Float16 h, l;
            split(v[i], h, l);
            hi[i] = h;
            lo[i] = l;
        }
        char* const to = a.direct + (size_t)matrix * a.out_bytes + at;
        *reinterpret_cast<halfx4*>(to) = hi;
        *reinterpret_cast<halfx4*>(to + 1024) = lo;
        if (mirror) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                char* const m = a.mirrored + (size_t)matrix * a.out_bytes + operand_at(p0 + i, q, 2 * a.qg);
                *reinterpret_cast<_Float16*>(m) = hi[i];
                *reinterpret_cast<_Float16*>(m + 1024) = lo[i];
            }
        }
    }
}

// Tile t of the upper triangle (with the diagonal), counted by columns: (row, column) with row <= column.
__device__ __forceinline__ void triangle(int t, int& row, int& col) {
    int c = (int)((sqrtf(8.0f * (float)t + 1.0f) - 1.0f) * 0.5f);
    while ((c + 1) * (c + 2) / 2 <= t) ++c;
    while (c * (c + 1) / 2 > t) --c;
    col = c;
    row = t - c * (c + 1) / 2;
}

// A workgroup takes 32 x 32 of C, each of its four waves a quarter of the reduction.  A and B are symmetric: only
// tiles on and above the diagonal are taken, and written both ways.
template <Product kind>
__global__ __launch_bounds__(256) void muon_product_small_kernel(ProductArgs a) {
    __shared__ float4 room[4][4][64];
    const int matrix = blockIdx.y, lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int tp, tq;
    if constexpr (kind == kGram || kind == kPoly) {
        triangle(blockIdx.x, tp, tq);
    } else {
        tp = blockIdx.x % a.pg;
        tq = blockIdx.x / a.pg;
    }
    const char* const p = a.p + (size_t)matrix * a.p_bytes + (size_t)tp * a.steps * kFragment + lane * 16;
    const char* const q = a.q + (size_t)matrix * a.q_bytes + (size_t)tq * a.steps * kFragment + lane * 16;
    floatx16 acc = {};
    const int per = (a.steps + 3) / 4, k1 = min(a.steps, (wave + 1) * per);
    for (int k = wave * per; k < k1; ++k) {
        const halfx8 ph = *reinterpret_cast<const halfx8*>(p + (size_t)k * kFragment);
        const halfx8 pl = *reinterpret_cast<const halfx8*>(p + (size_t)k * kFragment + 1024);
        const halfx8 qh = *reinterpret_cast<const halfx8*>(q + (size_t)k * kFragment);
        const halfx8 ql = *reinterpret_cast<const halfx8*>(q + (size_t)k * kFragment + 1024);
        acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(ph, ql, acc, 0, 0, 0);
        acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(pl, qh, acc, 0, 0, 0);
        acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(ph, qh, acc, 0, 0, 0);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) room[wave][j][lane] = make_float4(acc[4 * j], acc[4 * j + 1], acc[4 * j + 2], acc[4 * j + 3]);
    __syncthreads();
    float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        const float4 v = room[w][wave][lane];
        sum[0] += v.x; sum[1] += v.y; sum[2] += v.z; sum[3] += v.w;
    }
    const bool mirror = kind == kApply || tp != tq;
    write4<kind>(a, matrix, tp * 32 + 8 * wave + 4 * (lane >> 5), tq * 32 + (lane & 31), mirror, sum);
}

template <Product kind>
hipError_t launch_product(const ProductArgs& a, int count, hipStream_t s) {
    const int tiles = kind == kGram || kind == kPoly ? a.pg * (a.pg + 1) / 2 : a.pg * a.qg;
    hipLaunchKernelGGL((muon_product_small_kernel<kind>), dim3(tiles, count), dim3(256), 0, s, a);
    return hipGetLastError();
}

size_t rounded(size_t bytes) { return (bytes + 255) & ~(size_t)255; }

}  // namespace

size_t muon_workspace_bytes(int count, int rows, int cols) {
    const Shape s = shape_of(rows, cols);
    return rounded((size_t)count * norm_parts(rows, cols) * 8) + (size_t)count * (4 * s.x_bytes() + 2 * s.a_bytes());
}

hipError_t launch_muon(const MuonCall& c, hipStream_t s) {
    const Shape sh = shape_of(c.rows, c.cols);
    const bool update = c.weight.p != nullptr, tall = c.rows > c.cols;
    Front f{c.grad, c.momentum, update, c.nesterov, c.mu, c.rows, c.cols, norm_parts(c.rows, c.cols),
            static_cast<double*>(c.workspace)};
    char* at = static_cast<char*>(c.workspace) + rounded((size_t)c.count * f.parts * 8);
    char *x[2], *xt[2], *am, *bm;
    for (int i = 0; i < 2; ++i) {
        x[i] = at;
        at += c.count * sh.x_bytes();
        xt[i] = at;
        at += c.count * sh.x_bytes();
    }
    am = at;
    bm = at + c.count * sh.a_bytes();
    const dim3 fg(f.parts, c.count), pgrid((sh.mg + 1) / 2, (sh.ng + 1) / 2, c.count);
    const Pack pk{f, sh, tall, x[0], xt[0]};
    if (c.grad_bf16) {
        hipLaunchKernelGGL(muon_front_kernel<bf16_t>, fg, dim3(256), 0, s, f);
        hipLaunchKernelGGL(muon_pack_kernel<bf16_t>, pgrid, dim3(256), 0, s, pk);
    } else {
        hipLaunchKernelGGL(muon_front_kernel<float>, fg, dim3(256), 0, s, f);
        hipLaunchKernelGGL(muon_pack_kernel<float>, pgrid, dim3(256), 0, s, pk);
    }
    hipError_t e = hipGetLastError();
    for (int k = 0; k < c.steps && e == hipSuccess; ++k) {
        const int now = k & 1;
        ProductArgs g{};
        g.s = sh;
        g.p = g.q = x[now];
        g.p_bytes = g.q_bytes = sh.x_bytes();
        g.pg = g.qg = sh.mg;
        g.steps = 2 * sh.ng;
        g.direct = g.mirrored = am;
        g.out_bytes = sh.a_bytes();
        e = launch_product<kGram>(g, c.count, s);
        if (e != hipSuccess) break;
        g.p = g.q = g.old = am;
        g.p_bytes = g.q_bytes = sh.a_bytes();
        g.steps = 2 * sh.mg;
        g.direct = g.mirrored = bm;
        e = launch_product<kPoly>(g, c.count, s);
        if (e != hipSuccess) break;
        g.p = bm;
        g.q = g.old = xt[now];
        g.q_bytes = g.out_bytes = sh.x_bytes();
        g.qg = sh.ng;
        g.direct = xt[1 - now];
        g.mirrored = x[1 - now];
        if (k + 1 < c.steps) {
            e = launch_product<kApply>(g, c.count, s);
        } else {
            g.weight = c.weight;
            g.out = c.out;
            g.update = update;
            g.out_bf16 = c.out_bf16;
            g.tall = tall;
            g.keep = c.keep;
            g.rate = c.rate;
            e = launch_product<kLast>(g, c.count, s);
        }
    }
    return e;
}

}  // namespace rbmoe
