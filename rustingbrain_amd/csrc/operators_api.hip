// C ABI of the operators around the layer (see include/rbmoe.h): joining a sub-layer to the residual stream, and
// orthogonalised weight updates.  Checks of arguments and launches only; every call is enqueued on the context's
// stream, allocates nothing and waits for nothing, so it can be captured into a graph.
#include <cmath>
#include <cstdio>
#include <new>
#include <string>

#include "join_kernels.h"
#include "muon_kernels.h"
#include "rbmoe_context.h"

using namespace rbmoe;

struct rbmoe_join {
    rbmoe_ctx* ctx = nullptr;
    int cols = 0, dtype = 0, gate = 0;
    void* partial = nullptr;
    size_t partial_bytes = 0;
};

struct rbmoe_muon {
    rbmoe_ctx* ctx = nullptr;
    int count = 0, rows = 0, cols = 0;
    void* workspace = nullptr;
    size_t workspace_bytes = 0;
};

namespace {

constexpr int kMostJoinCols = 1 << 16, kMostJoinRows = 1 << 30, kMostMuonCount = 65535;

bool off_element(const void* p, int dtype) { return reinterpret_cast<uintptr_t>(p) % (dtype == RBMOE_BF16 ? 2 : 4) != 0; }

// What both directions of a join ask of their common arguments.
int join_problem(rbmoe_join* j, int32_t rows, const void* gate, float scale, float eps) {
    if (rows < 0) return fail(j->ctx, RBMOE_INVALID_INPUT, "the row count must not be negative");
    if (rows > kMostJoinRows) return fail(j->ctx, RBMOE_UNSUPPORTED, "more than 2^30 rows");
    if (rows > 0 && (j->gate != RBMOE_GATE_NONE) != (gate != nullptr))
        return fail(j->ctx, gate ? RBMOE_INVALID_INPUT : RBMOE_NULL_POINTER,
                    gate ? "this join was created without a gate" : "gate is NULL");
    if (!std::isfinite(scale)) return fail(j->ctx, RBMOE_INVALID_INPUT, "scale must be finite");
    if (!(eps >= 0.0f) || !std::isfinite(eps)) return fail(j->ctx, RBMOE_INVALID_INPUT, "eps must be finite and not negative");
    return RBMOE_OK;
}

}  // namespace

extern "C" {

int rbmoe_join_create(rbmoe_ctx* ctx, int32_t cols, int32_t dtype, int32_t gate, rbmoe_join** out) {
    if (!ctx || !out) return fail(ctx, RBMOE_NULL_POINTER, "ctx or out is NULL");
    *out = nullptr;
    if (cols <= 0) return fail(ctx, RBMOE_INVALID_CONFIG, "the row width must be positive");
    if (cols > kMostJoinCols) return fail(ctx, RBMOE_UNSUPPORTED, "rows of more than 65536 elements");
    if (dtype != RBMOE_F32 && dtype != RBMOE_BF16) return fail(ctx, RBMOE_INVALID_CONFIG, "rows must be f32 or bf16");
    if (gate != RBMOE_GATE_NONE && gate != RBMOE_GATE_CHANNEL && gate != RBMOE_GATE_ROW)
        return fail(ctx, RBMOE_INVALID_CONFIG, "the gate is none, by channel or by row");
    rbmoe_join* j = new (std::nothrow) rbmoe_join();
    if (!j) return fail(ctx, RBMOE_OUT_OF_MEMORY, "no host memory for the join");
    j->ctx = ctx;
    j->cols = cols;
    j->dtype = dtype;
    j->gate = gate;
    j->partial_bytes = (size_t)join_parts(cols) * 3 * cols * 4;
    if (const int rc = ctx_alloc(ctx, j->partial_bytes, "the join's partial sums", &j->partial)) {
        delete j;
        return rc;
    }
    ++ctx->refs;
    *out = j;
    return RBMOE_OK;
}

void rbmoe_join_destroy(rbmoe_join* j) {
    if (!j) return;
    (void)hipStreamSynchronize(j->ctx->stream);
    ctx_free(j->ctx, j->partial, j->partial_bytes);
    ctx_release(j->ctx);
    delete j;
}

int rbmoe_join_forward(rbmoe_join* j, int32_t rows, const void* x, const void* y, const uint8_t* valid, const float* post_weight,
                       const void* gate, float scale, const float* next_weight, float eps, void* out, void* normed) {
    if (!j) return fail(nullptr, RBMOE_NULL_POINTER, "join is NULL");
    rbmoe_ctx* ctx = j->ctx;
    if (const int rc = join_problem(j, rows, gate, scale, eps)) return rc;
    if (rows == 0) return RBMOE_OK;
    if (!x || !y || !out) return fail(ctx, RBMOE_NULL_POINTER, "x, y or out is NULL");
    if ((next_weight != nullptr) != (normed != nullptr))
        return fail(ctx, RBMOE_NULL_POINTER, "the norm in front of the next sub-layer needs both its weight and its rows");
    if (normed == out) return fail(ctx, RBMOE_INVALID_INPUT, "out and normed must not be the same rows");
    for (const void* p : {x, y, (const void*)out, (const void*)normed})
        if (off_element(p, j->dtype)) return fail(ctx, RBMOE_INVALID_INPUT, "rows must start at an element");
    if (off_element(gate, j->gate == RBMOE_GATE_ROW ? j->dtype : RBMOE_F32) || off_element(post_weight, RBMOE_F32) ||
        off_element(next_weight, RBMOE_F32))
        return fail(ctx, RBMOE_INVALID_INPUT, "weights and gate must start at an element");
    HIP_TRY(ctx, hipSetDevice(ctx->device));
    const JoinForward a{x, y, valid, post_weight, gate, next_weight, out, normed, rows, j->cols, j->gate, scale, eps};
    HIP_TRY(ctx, launch_join_forward(a, j->dtype == RBMOE_BF16, ctx->stream));
    return RBMOE_OK;
}

int rbmoe_join_backward(rbmoe_join* j, int32_t rows, const void* y, const void* out, const uint8_t* valid,
                        const float* post_weight, const void* gate, float scale, const float* next_weight, float eps,
                        const void* grad_out, const void* grad_normed, int32_t accumulate, void* grad_x, void* grad_y,
                        float* grad_post, void* grad_gate, float* grad_next) {
    if (!j) return fail(nullptr, RBMOE_NULL_POINTER, "join is NULL");
    rbmoe_ctx* ctx = j->ctx;
    if (const int rc = join_problem(j, rows, gate, scale, eps)) return rc;
    if (rows > 0) {
        if (!y || !grad_x || !grad_y) return fail(ctx, RBMOE_NULL_POINTER, "y, grad_x or grad_y is NULL");
        if ((next_weight != nullptr) != (grad_normed != nullptr) || (next_weight && !out))
            return fail(ctx, RBMOE_NULL_POINTER, "the norm in front of the next sub-layer needs its weight, its rows and their gradient");
        if (!grad_out && !grad_normed) return fail(ctx, RBMOE_NULL_POINTER, "grad_out is NULL and nothing follows");
        if (grad_x == grad_y) return fail(ctx, RBMOE_INVALID_INPUT, "grad_x and grad_y must not be the same rows");
    }
    if (grad_post && !post_weight && rows > 0) return fail(ctx, RBMOE_INVALID_INPUT, "grad_post without a norm behind the sub-layer");
    if (grad_next && !next_weight && rows > 0) return fail(ctx, RBMOE_INVALID_INPUT, "grad_next without a norm in front of the next sub-layer");
    if (grad_gate && j->gate == RBMOE_GATE_NONE) return fail(ctx, RBMOE_INVALID_INPUT, "this join was created without a gate");
    for (const void* p : {y, next_weight ? out : nullptr, grad_out, grad_normed, (const void*)grad_x, (const void*)grad_y})
        if (off_element(p, j->dtype)) return fail(ctx, RBMOE_INVALID_INPUT, "rows must start at an element");
    const int gate_dtype = j->gate == RBMOE_GATE_ROW ? j->dtype : RBMOE_F32;
    if (off_element(gate, gate_dtype) || off_element(grad_gate, gate_dtype) || off_element(post_weight, RBMOE_F32) ||
        off_element(next_weight, RBMOE_F32) || off_element(grad_post, RBMOE_F32) || off_element(grad_next, RBMOE_F32))
        return fail(ctx, RBMOE_INVALID_INPUT, "weights, gate and their gradients must start at an element");
    HIP_TRY(ctx, hipSetDevice(ctx->device));
    JoinBackward a{};
    a.y = y;
    a.out = next_weight ? out : nullptr;
    a.valid = valid;
    a.post = post_weight;
    a.gate = gate;
    a.next = next_weight;
    a.grad_out = grad_out;
    a.grad_normed = grad_normed;
    a.grad_x = grad_x;
    a.grad_y = grad_y;
    a.grad_post = grad_post;
    a.grad_gate = grad_gate;
    a.grad_next = grad_next;
    a.partial = static_cast<float*>(j->partial);
    a.rows = rows;
    a.cols = j->cols;
    a.gate_mode = j->gate;
    a.accumulate = accumulate != 0;
    a.scale = scale;
    a.eps = eps;
    HIP_TRY(ctx, launch_join_backward(a, j->dtype == RBMOE_BF16, ctx->stream));
    return RBMOE_OK;
}

int rbmoe_muon_create(rbmoe_ctx* ctx, int32_t count, int32_t rows, int32_t cols, rbmoe_muon** out) {
    if (!ctx || !out) return fail(ctx, RBMOE_NULL_POINTER, "ctx or out is NULL");
    *out = nullptr;
    if (count <= 0 || rows <= 0 || cols <= 0) return fail(ctx, RBMOE_INVALID_CONFIG, "count, rows and cols must be positive");
    if (count > kMostMuonCount || rows > kMostMuonSide || cols > kMostMuonSide)
        return fail(ctx, RBMOE_UNSUPPORTED, "more than 65535 matrices, or a matrix of more than 16384 rows or columns");
    rbmoe_muon* m = new (std::nothrow) rbmoe_muon();
    if (!m) return fail(ctx, RBMOE_OUT_OF_MEMORY, "no host memory for the updates");
    m->ctx = ctx;
    m->count = count;
    m->rows = rows;
    m->cols = cols;
    m->workspace_bytes = muon_workspace_bytes(count, rows, cols);
    if (const int rc = ctx_alloc(ctx, m->workspace_bytes, "the operands of the Newton-Schulz products", &m->workspace)) {
        delete m;
        return rc;
    }
    ++ctx->refs;
    *out = m;
    return RBMOE_OK;
}

void rbmoe_muon_destroy(rbmoe_muon* m) {
    if (!m) return;
    (void)hipStreamSynchronize(m->ctx->stream);
    ctx_free(m->ctx, m->workspace, m->workspace_bytes);
    ctx_release(m->ctx);
    delete m;
}

int rbmoe_orthogonalize(rbmoe_muon* m, const void* in, int32_t in_dtype, int32_t steps, void* out, int32_t out_dtype) {
    if (!m) return fail(nullptr, RBMOE_NULL_POINTER, "muon is NULL");
    rbmoe_ctx* ctx = m->ctx;
    if (!in || !out) return fail(ctx, RBMOE_NULL_POINTER, "in or out is NULL");
    for (const int dt : {in_dtype, out_dtype})
        if (dt != RBMOE_F32 && dt != RBMOE_BF16) return fail(ctx, RBMOE_INVALID_CONFIG, "matrices must be f32 or bf16");
    if (steps < 1 || steps > kMostMuonSteps) return fail(ctx, RBMOE_INVALID_CONFIG, "the number of steps must be between 1 and 64");
    if (off_element(in, in_dtype) || off_element(out, out_dtype)) return fail(ctx, RBMOE_INVALID_INPUT, "matrices must start at an element");
    HIP_TRY(ctx, hipSetDevice(ctx->device));
    MuonCall c;
    c.count = m->count;
    c.rows = m->rows;
    c.cols = m->cols;
    c.steps = steps;
    const size_t elements = (size_t)m->rows * m->cols;
    c.grad = {in, elements, m->cols};
    c.grad_bf16 = in_dtype == RBMOE_BF16;
    c.out = {out, elements, m->cols};
    c.out_bf16 = out_dtype == RBMOE_BF16;
    c.workspace = m->workspace;
    HIP_TRY(ctx, launch_muon(c, ctx->stream));
    return RBMOE_OK;
}

int rbmoe_muon_step(rbmoe_muon* m, const void* grad, int32_t grad_dtype, float* momentum, float* weight, float lr,
                    float momentum_factor, float weight_decay, float update_scale, int32_t nesterov, int32_t steps) {
    if (!m) return fail(nullptr, RBMOE_NULL_POINTER, "muon is NULL");
    rbmoe_ctx* ctx = m->ctx;
    if (!grad || !momentum || !weight) return fail(ctx, RBMOE_NULL_POINTER, "grad, momentum or weight is NULL");
    if (grad_dtype != RBMOE_F32 && grad_dtype != RBMOE_BF16) return fail(ctx, RBMOE_INVALID_CONFIG, "gradients must be f32 or bf16");
    if (const char* problem = muon_settings_problem(lr, momentum_factor, weight_decay, update_scale, steps))
        return fail(ctx, RBMOE_INVALID_CONFIG, problem);
    if (off_element(grad, grad_dtype) || off_element(momentum, RBMOE_F32) || off_element(weight, RBMOE_F32))
        return fail(ctx, RBMOE_INVALID_INPUT, "matrices must start at an element");
    if (momentum == weight || grad == momentum || grad == weight)
        return fail(ctx, RBMOE_INVALID_INPUT, "grad, momentum and weight must be three arrays");
    HIP_TRY(ctx, hipSetDevice(ctx->device));
    MuonCall c;
    c.count = m->count;
    c.rows = m->rows;
    c.cols = m->cols;
    c.steps = steps;
    const size_t elements = (size_t)m->rows * m->cols;
    c.grad = {grad, elements, m->cols};
    c.grad_bf16 = grad_dtype == RBMOE_BF16;
    c.momentum = {momentum, elements, m->cols};
    c.weight = {weight, elements, m->cols};
    c.mu = momentum_factor;
    c.keep = 1.0f - lr * weight_decay;
    c.rate = lr * muon_scale(update_scale, m->rows, m->cols);
    c.nesterov = nesterov != 0;
    c.workspace = m->workspace;
    HIP_TRY(ctx, launch_muon(c, ctx->stream));
    return RBMOE_OK;
}

// Which kernel takes a product (0: A, 1: B, 2: X) of a call: for tests (no GPU needed).
int rbmoe_internal_muon_tile(int32_t count, int32_t rows, int32_t cols, int32_t product) {
    return static_cast<int>(muon_tile(count, rows, cols, product));
}

}  // extern "C"
