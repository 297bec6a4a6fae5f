// Launches of join_kernels.hip.
#pragma once

#include <hip/hip_runtime.h>

#include <stddef.h>
#include <stdint.h>

#include "../../include/rbmoe.h"
#include "rbmoe_device.h"

namespace rbmoe {

// Row arrays are [rows, cols] of one type (f32 or bf16), parameters [cols] f32, a gate by channel [cols] f32 and by row like
// the row arrays.  `out` may be `x`, `normed` may be `y`, and a gradient of an input may lie where the gradient it is made
// from lies (the same addresses exactly).
struct JoinForward {
    const void* x;
    const void* y;
    const uint8_t* valid;  // [rows] or null: rows with 0 take y as zero
    const float* post;     // or null: no norm behind the sub-layer
    const void* gate;
    const float* next;     // or null: `normed` is not written
    void* out;
    void* normed;
    int rows, cols, gate_mode;
    float scale, eps;
};
struct JoinBackward {
    const void* y;
    const void* out;          // read with `next` only
    const uint8_t* valid;
    const float* post;
    const void* gate;
    const float* next;
    const void* grad_out;     // or null: zero
    const void* grad_normed;  // read with `next` only
    void* grad_x;             // or null
    void* grad_y;
    float* grad_post;         // these three: or null
    void* grad_gate;
    float* grad_next;
    float* partial;           // [join_parts(cols)][3][cols]
    int rows, cols, gate_mode, accumulate;
    float scale, eps;
};
int join_parts(int cols);  // workgroups of a backward launch at most
hipError_t launch_join_forward(const JoinForward& a, bool bf16, hipStream_t s);
hipError_t launch_join_backward(const JoinBackward& a, bool bf16, hipStream_t s);

}  // namespace rbmoe
