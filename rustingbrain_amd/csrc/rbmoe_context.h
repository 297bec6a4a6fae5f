// The context behind rbmoe_ctx and the error path that every C entry point shares.
#pragma once

#include <hip/hip_runtime.h>

#include <stddef.h>
#include <string>

#include "../../include/rbmoe.h"

struct rbmoe_ctx {
    int device = 0;
    hipStream_t own_stream = nullptr;
    hipStream_t stream = nullptr;
    // The backward pass runs the router's branch beside the weight gradients: a second stream (default
    // priority, like the first) forked from and joined to `stream` with two events.  Created on first use.
    hipStream_t side_stream = nullptr;
    hipEvent_t ev_fork = nullptr, ev_fork2 = nullptr, ev_join = nullptr, ev_tables = nullptr;
    // host calls: the routing of a forward is complete (recorded on `stream`), its tables are in host memory (recorded
    // on the side stream).  Created with the side stream.
    hipEvent_t ev_routed = nullptr, ev_fetched = nullptr;
    size_t budget_bytes = 0;
    size_t allocated = 0;
    void* static_scratch = nullptr;  // this device's copy of rbmoe_static_scratch (RBMOE_STATIC_SCRATCH_BYTES)
    std::string last_error;
    int refs = 1;  // the caller's handle + one per live layer or operator; torn down when the last one goes
};

namespace rbmoe {

// Records the message (on the context, where there is one, and for the calling thread) and returns `code`.
int fail(rbmoe_ctx* ctx, int code, const std::string& msg);
int hip_fail(rbmoe_ctx* ctx, hipError_t e, const char* what);

#define HIP_TRY(ctx, expr)                                         \
    do {                                                           \
        hipError_t _e = (expr);                                    \
        if (_e != hipSuccess) return hip_fail((ctx), _e, #expr);   \
    } while (0)

// One reference to the context less; the last one tears it down.
void ctx_release(rbmoe_ctx* ctx);

// Device memory of an operator's handle, counted against the context's budget before it is asked for.
int ctx_alloc(rbmoe_ctx* ctx, size_t bytes, const char* what, void** out);
void ctx_free(rbmoe_ctx* ctx, void* p, size_t bytes);

}  // namespace rbmoe
