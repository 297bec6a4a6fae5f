// A sub-layer joined to the residual stream, and its backward pass.
//
//   b      = N(y) * post          N(v)_j = v_j / sqrt(mean(v^2) + eps);  y itself without a norm behind the sub-layer
//   out    = x + scale * g * b
//   normed = N(out) * next        of the rows as they are stored in `out`, so that it equals a norm of its own behind this call
//
// Both directions are bound by memory: a row is read once, kept in registers in 32 bits, and everything that leaves it is
// written once.  A row belongs to one wave while it is short (no barrier, the sums go through lane permutations) and to a
// workgroup where it is long; rows beyond what registers hold are read again instead (the *_any kernels).
// The statistics and every sum are f32.  An output is rounded once, from f32.
//
// Backward, D = everything that reaches `out`:  with s = 1 / rms(out), t = 1 / rms(y), u = grad_normed * next
//   D         = grad_out + s (u - h (h . u) / d)     h = s out
//   grad_x    = D
//   grad_gate = scale * D * b             db = scale * g * D              v = db * post
//   grad_y    = t (v - n (n . v) / d)                n = t y
// (never by the cube of s or t alone: it leaves f32's range, below for an RMS above 4e12 and above for one below 1e-13, where both h and n are
// about one)
//   grad_post = sum_rows db * y * t       grad_next = sum_rows grad_normed * out * s
// us a call (bytes a second): forward 16384 x 1024 bf16 29.6 (4.5 TB/s; a copy of as much 5.2), 1 x 512 5.2, of which the launch is 2.8;
// backward 16384 x 1024 bf16 46.3 (4.3 TB/s), 1024 x 512 f32 9.2 (launches of 6 and 3).
// Each of the three parameter gradients is a sum over rows: a wave (or workgroup) takes every n-th row and keeps the sums of
// its columns in registers; workgroups then leave them in memory and a second, small launch adds them in a fixed order, so
// the same call gives the same bits.
#include "join_kernels.h"

#include <algorithm>

namespace rbmoe {

namespace {

// 16 bytes of a row, or of a parameter [d] (f32).  `A`: they start on a 16-byte boundary, and rows are whole pieces.  Otherwise they may start
// at any element (global memory takes 16-byte accesses at any address), and a row's last piece may have fewer elements: it is read as
// the 16 bytes that end with the row, and settle() moves it down once the loads are under way.  So these rows have V elements at least.
// What such a read holds of the lane before, which may be storing its piece in place, goes unused.
typedef uint32_t Any16 __attribute__((ext_vector_type(4), aligned(2), may_alias));
typedef uint32_t Any8 __attribute__((ext_vector_type(2), aligned(2), may_alias));
typedef uint32_t Any4 __attribute__((aligned(2), may_alias));
typedef uint16_t Any2 __attribute__((may_alias));

template <typename XT, bool A>
struct Piece {
    static constexpr int V = 16 / sizeof(XT);
    uint4 raw;
    __device__ __forceinline__ void zero() { raw = make_uint4(0, 0, 0, 0); }
    // p[0 .. n) of a row that ends at p + n, where n < V; nothing of it where n <= 0
    __device__ __forceinline__ void load(const XT* p, int n) {
        if (n <= 0) {
            zero();
        } else if constexpr (A) {
            raw = *reinterpret_cast<const uint4*>(p);
        } else {
            const Any16 v = *reinterpret_cast<const Any16*>(p - (V - min(n, V)));
            raw = make_uint4(v.x, v.y, v.z, v.w);
        }
    }
    // elements 0 .. n in their places, zeros behind them
    __device__ __forceinline__ void settle(int n) {
        if constexpr (!A) {
            if (n <= 0 || n >= V) return;
            const int away = V - n, words = sizeof(XT) == 2 ? away >> 1 : away;
            if (words & 2) raw = make_uint4(raw.z, raw.w, 0, 0);
            if (words & 1) raw = make_uint4(raw.y, raw.z, raw.w, 0);
            if (sizeof(XT) == 2 && (away & 1))
                raw = make_uint4(raw.x >> 16 | raw.y << 16, raw.y >> 16 | raw.z << 16, raw.z >> 16 | raw.w << 16, raw.w >> 16);
        }
    }
    __device__ __forceinline__ void widen(float (&v)[V]) const { Vec16<XT>::widen(raw, v); }
    // n > 0
    static __device__ __forceinline__ void store(XT* p, const float (&v)[V], int n) {
        uint4 o;
        if constexpr (sizeof(XT) == 2) o = make_uint4(pack2(v[0], v[1]), pack2(v[2], v[3]), pack2(v[4], v[5]), pack2(v[6], v[7]));
        else o = make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
        if constexpr (A) {
            *reinterpret_cast<uint4*>(p) = o;
        } else if (n >= V) {
            *reinterpret_cast<Any16*>(p) = Any16{o.x, o.y, o.z, o.w};
        } else {
            constexpr int W = 4 / sizeof(XT);  // elements of a word
            if (n & 2 * W) {
                *reinterpret_cast<Any8*>(p) = Any8{o.x, o.y};
                o.x = o.z, o.y = o.w;
                p += 2 * W;
            }
            if (n & W) {
                *reinterpret_cast<Any4*>(p) = o.x;
                o.x = o.y;
                p += W;
            }
            if constexpr (W == 2)
                if (n & 1) *reinterpret_cast<Any2*>(p) = (uint16_t)o.x;
        }
    }
};

// V values of a parameter at a column with n of the row's left (n > 0), and back
template <int V, bool A>
__device__ __forceinline__ void load_parameter(const float* p, float (&v)[V], int n) {
    Piece<float, A> a[V / 4];
#pragma unroll
    for (int q = 0; q < V / 4; ++q) a[q].load(p + 4 * q, A ? V : n - 4 * q);
#pragma unroll
    for (int q = 0; q < V / 4; ++q) {
        a[q].settle(n - 4 * q);
        float w[4];
        a[q].widen(w);
        v[4 * q] = w[0]; v[4 * q + 1] = w[1]; v[4 * q + 2] = w[2]; v[4 * q + 3] = w[3];
    }
}
template <int V, bool A>
__device__ __forceinline__ void store_parameter(float* p, const float (&v)[V], int n) {
#pragma unroll
    for (int q = 0; q < V / 4; ++q) {
        const float w[4] = {v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]};
        if (A || n > 4 * q) Piece<float, A>::store(p + 4 * q, w, n - 4 * q);
    }
}

// What the stored row holds for an f32 value.
template <typename XT>
__device__ __forceinline__ float as_stored(float v) {
    if constexpr (sizeof(XT) == 2) return bf16_bits_to_f32(f32_to_bf16_bits(v));
    return v;
}

__device__ __forceinline__ float wave_sum(float v) {
    return __uint_as_float(group_reduce(__float_as_uint(v), 64, [](uint32_t a, uint32_t b) {
        return __float_as_uint(__uint_as_float(a) + __uint_as_float(b));
    }));
}

// N sums over the G threads of a row, the same in all of them: G is a wave, or the whole workgroup (every thread of which
// then calls; `room`: 4 N floats that the next call of this function may overwrite at once - two are used in turn).
template <int G, int N>
__device__ __forceinline__ void row_sums(float (&s)[N], float* room) {
#pragma unroll
    for (int i = 0; i < N; ++i) s[i] = wave_sum(s[i]);
    if constexpr (G > 64) {
        constexpr int W = G / 64;
        const int wave = threadIdx.x >> 6;
        if ((threadIdx.x & 63) == 0)
#pragma unroll
            for (int i = 0; i < N; ++i) room[i * W + wave] = s[i];
        __syncthreads();
#pragma unroll
        for (int i = 0; i < N; ++i) {
            float t = room[i * W];
#pragma unroll
            for (int w = 1; w < W; ++w) t += room[i * W + w];
            s[i] = t;
        }
    }
}

__device__ __forceinline__ float inverse_rms(float sum_of_squares, int d, float eps) {
    return 1.0f / sqrtf(sum_of_squares / (float)d + eps);
}

// ---- forward -----------------------------------------------------------------------------------
// A launch holds 2^32 threads a dimension at most, which is fewer than 2^30 rows take: the workgroups of a forward launch lie in two.
__device__ __forceinline__ int row_block() { return blockIdx.y * gridDim.x + blockIdx.x; }
dim3 row_grid(int blocks) {
    const int wide = std::min(blocks, 1 << 20);
    return dim3(wide, (blocks + wide - 1) / wide);
}

template <typename XT, bool A, int P, int G>
__global__ __launch_bounds__(256) void join_forward_kernel(JoinForward a) {
    constexpr int V = Piece<XT, A>::V, RPB = 256 / G;  // elements of a piece, rows of a workgroup
    __shared__ float room[2][4];
    const int lane = threadIdx.x % G, d = a.cols;
    const int row = row_block() * RPB + threadIdx.x / G;
    if (row >= a.rows) return;  // (a whole wave's rows, or the whole workgroup's)
    const size_t at = (size_t)row * d;
    const XT* const x = static_cast<const XT*>(a.x) + at;
    const XT* const y = static_cast<const XT*>(a.y) + at;
    const bool live = a.valid == nullptr || a.valid[row] != 0;
    Piece<XT, A> yr[P], xr[P];
#pragma unroll
    for (int p = 0; p < P; ++p) {
        const int c = (p * G + lane) * V;
        yr[p].load(y + c, live ? d - c : 0);
        xr[p].load(x + c, d - c);
    }
#pragma unroll
    for (int p = 0; p < P; ++p) {
        const int n = d - (p * G + lane) * V;
        yr[p].settle(n);
        xr[p].settle(n);
    }
    float factor = 1.0f;
    if (a.post) {
        float s[1] = {0.0f};
#pragma unroll
        for (int p = 0; p < P; ++p) {
            float v[V];
            yr[p].widen(v);
#pragma unroll
            for (int i = 0; i < V; ++i) s[0] = fmaf(v[i], v[i], s[0]);
        }
        row_sums<G>(s, room[0]);
        factor = inverse_rms(s[0], d, a.eps);
    }
    float out[P][V], s2[1] = {0.0f};
#pragma unroll
    for (int p = 0; p < P; ++p) {
        const int c = (p * G + lane) * V;
        float xv[V], b[V];
        xr[p].widen(xv);
        yr[p].widen(b);
        if (c < d) {
            if (live) {
                if (a.post) {
                    float w[V];
                    load_parameter<V, A>(a.post + c, w, d - c);
#pragma unroll
                    for (int i = 0; i < V; ++i) b[i] = b[i] * factor * w[i];
                }
                if (a.gate_mode == RBMOE_GATE_CHANNEL) {
                    float g[V];
                    load_parameter<V, A>(static_cast<const float*>(a.gate) + c, g, d - c);
#pragma unroll
                    for (int i = 0; i < V; ++i) b[i] *= g[i];
                } else if (a.gate_mode == RBMOE_GATE_ROW) {
                    Piece<XT, A> gr;
                    gr.load(static_cast<const XT*>(a.gate) + at + c, d - c);
                    gr.settle(d - c);
                    float g[V];
                    gr.widen(g);
#pragma unroll
                    for (int i = 0; i < V; ++i) b[i] *= g[i];
                }
            }
#pragma unroll
            for (int i = 0; i < V; ++i) out[p][i] = live ? as_stored<XT>(fmaf(a.scale, b[i], xv[i])) : xv[i];
            Piece<XT, A>::store(static_cast<XT*>(a.out) + at + c, out[p], d - c);
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i) out[p][i] = 0.0f;
        }
#pragma unroll
        for (int i = 0; i < V; ++i) s2[0] = fmaf(out[p][i], out[p][i], s2[0]);
    }
    if (!a.next) return;
    row_sums<G>(s2, room[1]);
    const float f2 = inverse_rms(s2[0], d, a.eps);
#pragma unroll
    for (int p = 0; p < P; ++p) {
        const int c = (p * G + lane) * V;
        if (c < d) {
            float w[V];
            load_parameter<V, A>(a.next + c, w, d - c);
#pragma unroll
            for (int i = 0; i < V; ++i) w[i] = out[p][i] * f2 * w[i];
            Piece<XT, A>::store(static_cast<XT*>(a.normed) + at + c, w, d - c);
        }
    }
}

// Rows of any width: a workgroup a row, read again for each step.  A thread reads back only what it wrote itself.
template <typename XT>
__global__ __launch_bounds__(256) void join_forward_any_kernel(JoinForward a) {
    __shared__ float room[2][4];
    const int d = a.cols, row = row_block();
    if (row >= a.rows) return;
    const size_t at = (size_t)row * d;
    const XT* const x = static_cast<const XT*>(a.x) + at;
    const XT* const y = static_cast<const XT*>(a.y) + at;
    XT* const out = static_cast<XT*>(a.out) + at;
    const bool live = a.valid == nullptr || a.valid[row] != 0;
    float factor = 1.0f;
    if (a.post) {
        float s[1] = {0.0f};
        for (int c = threadIdx.x; live && c < d; c += 256) {
            const float v = to_f32(y[c]);
            s[0] = fmaf(v, v, s[0]);
        }
        row_sums<256>(s, room[0]);
        factor = inverse_rms(s[0], d, a.eps);
    }
    float s2[1] = {0.0f};
    for (int c = threadIdx.x; c < d; c += 256) {
        float o = to_f32(x[c]);
        if (live) {
            float b = to_f32(y[c]);
            if (a.post) b = b * factor * a.post[c];
            if (a.gate_mode == RBMOE_GATE_CHANNEL) b *= static_cast<const float*>(a.gate)[c];
            else if (a.gate_mode == RBMOE_GATE_ROW) b *= to_f32(static_cast<const XT*>(a.gate)[at + c]);
            o = as_stored<XT>(fmaf(a.scale, b, o));
        }
        out[c] = from_f32<XT>(o);
        s2[0] = fmaf(o, o, s2[0]);
    }
    if (!a.next) return;
    row_sums<256>(s2, room[1]);
    const float f2 = inverse_rms(s2[0], d, a.eps);
    for (int c = threadIdx.x; c < d; c += 256)
        static_cast<XT*>(a.normed)[at + c] = from_f32<XT>(to_f32(out[c]) * f2 * a.next[c]);
}

// ---- backward ----------------------------------------------------------------------------------
// Where the sums over rows go: workgroup b of n leaves its own in partial[b][which][d]; with one workgroup they are final.
__device__ __forceinline__ float* sum_target(const JoinBackward& a, int which) {
    return which == 0 ? a.grad_post : which == 1 ? (a.gate_mode == RBMOE_GATE_CHANNEL ? static_cast<float*>(a.grad_gate) : nullptr)
                                                 : a.grad_next;
}

template <typename XT, bool A, int P, int G>
__global__ __launch_bounds__(256) void join_backward_kernel(JoinBackward a) {
    constexpr int V = Piece<XT, A>::V, RPB = 256 / G;
    __shared__ float room[2][12];
    const int lane = threadIdx.x % G, d = a.cols;
    const float inv_d = 1.0f / (float)d;
    const bool has_post = a.post != nullptr, has_next = a.next != nullptr;
    float sums[3][P][V];
#pragma unroll
    for (int k = 0; k < 3; ++k)
#pragma unroll
        for (int p = 0; p < P; ++p)
#pragma unroll
            for (int i = 0; i < V; ++i) sums[k][p][i] = 0.0f;
    // the parameters of the thread's columns stay in registers from row to row
    float next[P][V], post[P][V], gate[P][V];
#pragma unroll
    for (int p = 0; p < P; ++p) {
        const int c = (p * G + lane) * V;
#pragma unroll
        for (int i = 0; i < V; ++i) next[p][i] = 0.0f, post[p][i] = gate[p][i] = 1.0f;
        if (c >= d) continue;
        if (has_next) load_parameter<V, A>(a.next + c, next[p], d - c);
        if (has_post) load_parameter<V, A>(a.post + c, post[p], d - c);
        if (a.gate_mode == RBMOE_GATE_CHANNEL) load_parameter<V, A>(static_cast<const float*>(a.gate) + c, gate[p], d - c);
    }
    for (int row = blockIdx.x * RPB + threadIdx.x / G; row < a.rows; row += gridDim.x * RPB) {
        const size_t at = (size_t)row * d;
        const bool live = a.valid == nullptr || a.valid[row] != 0;
        Piece<XT, A> yr[P], rr[P], gr[P], nr[P];
#pragma unroll
        for (int p = 0; p < P; ++p) {
            const int c = (p * G + lane) * V;
            yr[p].load(static_cast<const XT*>(a.y) + at + c, live ? d - c : 0);
            gr[p].load(static_cast<const XT*>(a.grad_out) + at + c, a.grad_out ? d - c : 0);
            rr[p].load(static_cast<const XT*>(a.out) + at + c, has_next ? d - c : 0);
            nr[p].load(static_cast<const XT*>(a.grad_normed) + at + c, has_next ? d - c : 0);
        }
#pragma unroll
        for (int p = 0; p < P; ++p) {
            const int n = d - (p * G + lane) * V;
            yr[p].settle(n);
            gr[p].settle(n);
            rr[p].settle(n);
            nr[p].settle(n);
        }
        float s[3] = {0.0f, 0.0f, 0.0f};  // out^2, out . u, y^2
#pragma unroll
        for (int p = 0; p < P; ++p) {
            float yv[V];
            yr[p].widen(yv);
#pragma unroll
            for (int i = 0; i < V; ++i) s[2] = fmaf(yv[i], yv[i], s[2]);
            if (has_next) {
                float rv[V], nv[V];
                rr[p].widen(rv);
                nr[p].widen(nv);
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    s[0] = fmaf(rv[i], rv[i], s[0]);
                    s[1] = fmaf(rv[i], nv[i] * next[p][i], s[1]);
                }
            }
        }
        row_sums<G>(s, room[0]);
        const float k2 = has_next ? inverse_rms(s[0], d, a.eps) : 0.0f;
        const float dot2 = s[1] * k2 * inv_d;
        const float k1 = has_post ? inverse_rms(s[2], d, a.eps) : 1.0f;
        float D[P][V], yv_dot[1] = {0.0f};
#pragma unroll
        for (int p = 0; p < P; ++p) {
            const int c = (p * G + lane) * V;
            gr[p].widen(D[p]);
            if (c >= d) continue;
            if (has_next) {
                float rv[V], nv[V];
                rr[p].widen(rv);
                nr[p].widen(nv);
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const float h = rv[i] * k2;
                    D[p][i] += k2 * (nv[i] * next[p][i] - h * dot2);
                    if (live) sums[2][p][i] = fmaf(nv[i], h, sums[2][p][i]);
                }
            }
            if (a.grad_x) Piece<XT, A>::store(static_cast<XT*>(a.grad_x) + at + c, D[p], d - c);
            // from here on D is the gradient of what the gate let through, then of the norm's output
            float yv[V], g[V];
            yr[p].widen(yv);
#pragma unroll
            for (int i = 0; i < V; ++i) g[i] = gate[p][i];
            if (a.gate_mode == RBMOE_GATE_ROW && live) {
                Piece<XT, A> q;
                q.load(static_cast<const XT*>(a.gate) + at + c, d - c);
                q.settle(d - c);
                q.widen(g);
            }
            float dg[V];
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float n = yv[i] * k1, e = live ? a.scale * D[p][i] : 0.0f;
                dg[i] = live ? e * (n * post[p][i]) : 0.0f;
                const float db = e * g[i];
                sums[0][p][i] = live ? fmaf(db, n, sums[0][p][i]) : sums[0][p][i];
                sums[1][p][i] += dg[i];
                D[p][i] = has_post ? db * post[p][i] : db;
                yv_dot[0] = fmaf(yv[i], D[p][i], yv_dot[0]);
            }
            if (a.gate_mode == RBMOE_GATE_ROW && a.grad_gate) Piece<XT, A>::store(static_cast<XT*>(a.grad_gate) + at + c, dg, d - c);
        }
        float dot1 = 0.0f;
        if (has_post) {
            row_sums<G>(yv_dot, room[1]);
            dot1 = yv_dot[0] * k1 * inv_d;
        }
#pragma unroll
        for (int p = 0; p < P; ++p) {
            const int c = (p * G + lane) * V;
            if (c >= d) continue;
            float yv[V];
            yr[p].widen(yv);
#pragma unroll
            for (int i = 0; i < V; ++i)  // (without a norm it does not depend on y, which may be infinite)
                yv[i] = !live ? 0.0f : has_post ? k1 * (D[p][i] - yv[i] * k1 * dot1) : D[p][i];
            Piece<XT, A>::store(static_cast<XT*>(a.grad_y) + at + c, yv, d - c);
        }
        if constexpr (G > 64) __syncthreads();  // `room` is written again
    }
    // the sums of the workgroup: where it has several waves, added in wave order, every thread some columns
    const bool add = gridDim.x == 1 && a.accumulate;
    auto place = [&](int k) { return gridDim.x == 1 ? sum_target(a, k) : a.partial + ((size_t)blockIdx.x * 3 + k) * d; };
    if constexpr (RPB > 1) {
        __shared__ __align__(16) float stage[3][RPB][P * G * V];
#pragma unroll
        for (int k = 0; k < 3; ++k)
            if (sum_target(a, k))  // uniform
#pragma unroll
                for (int p = 0; p < P; ++p) store_parameter<V, true>(stage[k][threadIdx.x / G] + (p * G + lane) * V, sums[k][p], V);
        __syncthreads();
#pragma unroll
        for (int k = 0; k < 3; ++k) {
            if (!sum_target(a, k)) continue;
            float* const dst = place(k);
            for (int c = threadIdx.x; c < d; c += 256) {
                float v = stage[k][0][c];
#pragma unroll
                for (int w = 1; w < RPB; ++w) v += stage[k][w][c];
                dst[c] = v + (add ? dst[c] : 0.0f);
            }
        }
    } else {
#pragma unroll
        for (int k = 0; k < 3; ++k) {
            if (!sum_target(a, k)) continue;
            float* const dst = place(k);
#pragma unroll
            for (int p = 0; p < P; ++p) {
                const int c = (p * G + lane) * V;
                if (c >= d) continue;
                if (add) {
                    float before[V];
                    load_parameter<V, false>(dst + c, before, d - c);
#pragma unroll
                    for (int i = 0; i < V; ++i) sums[k][p][i] += before[i];
                }
                store_parameter<V, false>(dst + c, sums[k][p], d - c);
            }
        }
    }
}

// Rows of any width: a workgroup takes every n-th row and reads it again for each step; its sums over rows lie in memory of
// its own (partial[b]), where a thread adds only to columns of its own.
template <typename XT>
__global__ __launch_bounds__(256) void join_backward_any_kernel(JoinBackward a) {
    __shared__ float room[2][12];
    const int d = a.cols;
    const float inv_d = 1.0f / (float)d;
    const bool has_post = a.post != nullptr, has_next = a.next != nullptr;
    float* const mine = a.partial + (size_t)blockIdx.x * 3 * d;
    for (int c = threadIdx.x; c < d; c += 256) mine[c] = mine[d + c] = mine[2 * (size_t)d + c] = 0.0f;
    for (int row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const size_t at = (size_t)row * d;
        const bool live = a.valid == nullptr || a.valid[row] != 0;
        const XT* const y = static_cast<const XT*>(a.y) + at;
        const XT* const r = has_next ? static_cast<const XT*>(a.out) + at : nullptr;
        const XT* const go = a.grad_out ? static_cast<const XT*>(a.grad_out) + at : nullptr;
        const XT* const gn = has_next ? static_cast<const XT*>(a.grad_normed) + at : nullptr;
        float s[3] = {0.0f, 0.0f, 0.0f};
        for (int c = threadIdx.x; c < d; c += 256) {
            const float yv = live ? to_f32(y[c]) : 0.0f;
            s[2] = fmaf(yv, yv, s[2]);
            if (has_next) {
                const float rv = to_f32(r[c]);
                s[0] = fmaf(rv, rv, s[0]);
                s[1] = fmaf(rv, to_f32(gn[c]) * a.next[c], s[1]);
            }
        }
        row_sums<256>(s, room[0]);
        const float k2 = has_next ? inverse_rms(s[0], d, a.eps) : 0.0f;
        const float dot2 = s[1] * k2 * inv_d;
        const float k1 = has_post ? inverse_rms(s[2], d, a.eps) : 1.0f;
        auto total = [&](int c) {  // D
            float v = go ? to_f32(go[c]) : 0.0f;
            if (has_next) v += k2 * (to_f32(gn[c]) * a.next[c] - to_f32(r[c]) * k2 * dot2);
            return v;
        };
        auto gate = [&](int c) {
            return a.gate_mode == RBMOE_GATE_CHANNEL ? static_cast<const float*>(a.gate)[c]
                   : a.gate_mode == RBMOE_GATE_ROW   ? to_f32(static_cast<const XT*>(a.gate)[at + c])
                                                     : 1.0f;
        };
        float dot[1] = {0.0f};
        if (has_post) {
            for (int c = threadIdx.x; live && c < d; c += 256)
                dot[0] = fmaf(to_f32(y[c]), a.scale * total(c) * gate(c) * a.post[c], dot[0]);
            row_sums<256>(dot, room[1]);
        }
        const float dot1 = has_post ? dot[0] * k1 * inv_d : 0.0f;
        for (int c = threadIdx.x; c < d; c += 256) {
            const float D = total(c);
            float dy = 0.0f, dg = 0.0f;
            if (live) {
                const float yv = to_f32(y[c]), n = yv * k1, w = has_post ? a.post[c] : 1.0f, e = a.scale * D, db = e * gate(c);
                dg = e * (n * w);
                mine[c] += db * n;
                mine[d + c] += dg;
                dy = has_post ? k1 * (db * w - n * dot1) : db;
                if (has_next) mine[2 * (size_t)d + c] = fmaf(to_f32(gn[c]), to_f32(r[c]) * k2, mine[2 * (size_t)d + c]);
            }
            if (a.gate_mode == RBMOE_GATE_ROW && a.grad_gate) static_cast<XT*>(a.grad_gate)[at + c] = from_f32<XT>(dg);
            if (a.grad_x) static_cast<XT*>(a.grad_x)[at + c] = from_f32<XT>(D);
            static_cast<XT*>(a.grad_y)[at + c] = from_f32<XT>(dy);
        }
        __syncthreads();  // `room` is written again
    }
}

// The workgroups' sums, added in the order of the workgroups: 32 columns a workgroup, 16 threads a column, each over every
// 16th workgroup with its loads under way together.  us a backward call of 1024 x 512 f32 / 3001 x 760 bf16 / 16384 x 1024 bf16: 8 threads 9.7 / 15.5 /
// 48.0, 16 9.2 / 14.5 / 46.3, 32 10.6 / 15.1 / 46.5.
constexpr int kSumSlices = 16;
__global__ __launch_bounds__(32 * kSumSlices) void join_sums_kernel(JoinBackward a, int parts) {
    float* const dst = sum_target(a, blockIdx.y);
    if (!dst) return;
    __shared__ float room[kSumSlices][33];
    const int d = a.cols, c = blockIdx.x * 32 + (threadIdx.x & 31), slice = threadIdx.x >> 5;
    float s = 0.0f;
    if (c < d) {
        const float* src = a.partial + (size_t)blockIdx.y * d + c;
#pragma unroll 16
        for (int b = slice; b < parts; b += kSumSlices) s += src[(size_t)b * 3 * d];
    }
    room[slice][threadIdx.x & 31] = s;
    __syncthreads();
    if (slice == 0 && c < d) {
#pragma unroll
        for (int w = 1; w < kSumSlices; ++w) s += room[w][threadIdx.x & 31];
        dst[c] = s + (a.accumulate ? dst[c] : 0.0f);
    }
}

uintptr_t address(const void* p) { return reinterpret_cast<uintptr_t>(p); }

// Whether rows of `cols` elements are whole pieces on 16-byte boundaries, and the parameters lie on them too.
bool on_pieces(int cols, int size, uintptr_t rows_at, uintptr_t parameters_at) {
    return (size_t)cols * size % 16 == 0 && rows_at % 16 == 0 && parameters_at % 16 == 0;
}

// f(A, P, G) as integral constants for rows of `cols` elements, or `any()` where registers do not hold them.  Rows off 16 bytes by whole
// vectors too, against two (bf16) or one element an access, us forward / backward: 1533 x 1365 f32 8.7 / 25.3 -> 7.6 / 24.3, 2000 x 1365
// bf16 10.2 / 41.6 -> 7.8 / 23.1, 2000 x 2047 bf16 13.5 / 48.7 -> 9.6 / 25.2; 1000 x 766 bf16 6.3 / 14.7 -> 6.0 / 15.6,
// 4000 x 766 8.7 / 20.6 -> 8.7 / 22.9.  (Even bf16 widths off 16 bytes lose 6 to 11 % in the backward pass where odd ones gain 1.8 times; there is no
// third form of the kernels for those alone.)  A wave takes a
// row of up to 16 elements a lane, a workgroup one of up to 32 a thread.  us a call, rows of 2048 bf16 by a wave / by a
// workgroup: 200 rows 6.4 / 4.9, 2000 rows 9.2 / 8.0; rows of 768: 203 rows 4.9 / 4.9, 2000 rows 5.4 / 5.6, of 1024, 4096 rows 7.8 / 8.8.
// Backward, 32 elements a thread (up to 423 registers, one wave a SIMD, nothing in memory) against rows read again: 1 x 5000 bf16
// 34 -> 7.2, 2000 x 5001 250 -> 60, 4096 x 8192 964 -> 113, 4096 x 8192 f32 842 -> 184.
template <typename XT, typename F, typename N>
hipError_t with_shape(int cols, bool whole, F&& f, N&& any) {
    constexpr int V = 16 / sizeof(XT);
    auto pick = [&](auto pieces) -> hipError_t {
        const int wave = (cols + 64 * V - 1) / (64 * V), group = (cols + 256 * V - 1) / (256 * V);
        if (cols < V) return any();  // no whole piece in a row
        typedef std::integral_constant<int, 1> One;
        typedef std::integral_constant<int, 2> Two;
        typedef std::integral_constant<int, 4> Four;
        typedef std::integral_constant<int, 8> Eight;
        typedef std::integral_constant<int, 64> Wave;
        typedef std::integral_constant<int, 256> Group;
        if (wave <= 1) return f(pieces, One{}, Wave{});
        if (wave <= 2) return f(pieces, Two{}, Wave{});
        if constexpr (4 * V <= 16)
            if (wave <= 4) return f(pieces, Four{}, Wave{});
        if (group <= 1) return f(pieces, One{}, Group{});
        if (group <= 2) return f(pieces, Two{}, Group{});
        if (group <= 4) return f(pieces, Four{}, Group{});
        if constexpr (8 * V <= 32)
            if (group <= 8) return f(pieces, Eight{}, Group{});
        return any();
    };
    return whole ? pick(std::true_type{}) : pick(std::false_type{});
}

// Workgroups of a backward launch at most: two a compute unit, which is what their registers allow up to 16 elements a thread, and whose sums (12 bytes a column) are
// written and read again.  16384 x 1024 bf16: 512 48 us, 768 65.
constexpr int kMostParts = 512;

hipError_t add_parts(const JoinBackward& a, int parts, hipStream_t s) {
    if (!a.grad_post && !a.grad_next && !(a.gate_mode == RBMOE_GATE_CHANNEL && a.grad_gate)) return hipSuccess;
    hipLaunchKernelGGL(join_sums_kernel, dim3((a.cols + 31) / 32, 3), dim3(32 * kSumSlices), 0, s, a, parts);
    return hipGetLastError();
}

template <typename XT>
hipError_t forward(const JoinForward& a, hipStream_t s) {
    const uintptr_t rows = address(a.x) | address(a.y) | address(a.out) | address(a.normed) |
                           (a.gate_mode == RBMOE_GATE_ROW ? address(a.gate) : 0);
    const uintptr_t parameters = address(a.post) | address(a.next) | (a.gate_mode == RBMOE_GATE_CHANNEL ? address(a.gate) : 0);
    return with_shape<XT>(
        a.cols, on_pieces(a.cols, sizeof(XT), rows, parameters),
        [&](auto whole, auto p, auto g) {
            constexpr int P = decltype(p)::value, G = decltype(g)::value, RPB = 256 / G;
            hipLaunchKernelGGL((join_forward_kernel<XT, decltype(whole)::value, P, G>), row_grid((a.rows + RPB - 1) / RPB), dim3(256), 0, s, a);
            return hipGetLastError();
        },
        [&] {
            hipLaunchKernelGGL((join_forward_any_kernel<XT>), row_grid(a.rows), dim3(256), 0, s, a);
            return hipGetLastError();
        });
}

template <typename XT>
hipError_t backward(const JoinBackward& a, hipStream_t s) {
    const uintptr_t rows = address(a.y) | address(a.out) | address(a.grad_out) | address(a.grad_normed) | address(a.grad_x) |
                           address(a.grad_y) | (a.gate_mode == RBMOE_GATE_ROW ? address(a.gate) | address(a.grad_gate) : 0);
    const uintptr_t parameters = address(a.post) | address(a.next) | (a.gate_mode == RBMOE_GATE_CHANNEL ? address(a.gate) : 0);
    const int most = join_parts(a.cols);
    int parts = 0;
    bool final = false;
    hipError_t e = with_shape<XT>(
        a.cols, on_pieces(a.cols, sizeof(XT), rows, parameters),
        [&](auto whole, auto p, auto g) {
            constexpr int P = decltype(p)::value, G = decltype(g)::value, RPB = 256 / G;
            // one workgroup a compute unit where a thread's 32 elements leave room for no second: 2000 x 5001 bf16 68.6 -> 59.7 us,
            // 4096 x 8192 122 -> 113, 300 x 8190 f32 41 -> 33
            const int limit = P * 16 / (int)sizeof(XT) >= 32 ? std::min(most, 256) : most;
            // as many rows for every wave (or workgroup) as the busiest has
            const int turns = (a.rows + RPB - 1) / RPB, each = (turns + limit - 1) / limit;
            parts = (turns + each - 1) / each;
            final = parts == 1;
            hipLaunchKernelGGL((join_backward_kernel<XT, decltype(whole)::value, P, G>), dim3(parts), dim3(256), 0, s, a);
            return hipGetLastError();
        },
        [&] {
            parts = std::min(a.rows, most);
            hipLaunchKernelGGL((join_backward_any_kernel<XT>), dim3(parts), dim3(256), 0, s, a);
            return hipGetLastError();
        });
    return e != hipSuccess || final ? e : add_parts(a, parts, s);
}

}  // namespace

int join_parts(int cols) { return std::max(32, std::min(kMostParts, (1 << 22) / std::max(cols, 1))); }

hipError_t launch_join_forward(const JoinForward& a, bool bf16, hipStream_t s) {
    if (a.rows == 0) return hipSuccess;
    return bf16 ? forward<bf16_t>(a, s) : forward<float>(a, s);
}

hipError_t launch_join_backward(const JoinBackward& a, bool bf16, hipStream_t s) {
    if (a.rows == 0) return a.accumulate ? hipSuccess : add_parts(a, 0, s);  // (sums over no rows: zero)
    return bf16 ? backward<bf16_t>(a, s) : backward<float>(a, s);
}

}  // namespace rbmoe
