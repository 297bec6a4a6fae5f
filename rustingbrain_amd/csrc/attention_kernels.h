// Launches of attention_kernels.hip.
#pragma once

#include <hip/hip_runtime.h>

#include <stddef.h>
#include <stdint.h>

#include "../../include/rbmoe.h"
#include "rbmoe_device.h"

namespace rbmoe {

constexpr int kMostHeadDim = 128;

// Rows are [rows, heads, head_dim], a row's heads contiguous, rows `*_stride` elements apart; out and grad_out without gaps, a
// gradient of an input like its input.  lse is [heads, query_rows] f32.
struct AttentionCall {
    const void* q;
    const void* k;
    const void* v;
    void* out;
    float* lse;        // or null (forward)
    const int32_t* query_begin;
    const int32_t* query_count;
    const int32_t* key_begin;
    const int32_t* key_count;
    long long q_stride, k_stride, v_stride;
    int sequences, query_rows, key_rows, longest_queries, longest_keys;
    int heads, kv_heads, head_dim, causal;
    float scale;
    // backward
    const void* grad_out;
    void* grad_q;
    void* grad_k;
    void* grad_v;
    float* delta;  // [2][heads, query_rows], references of the exponents and deltas: written by the queries' gradients, read by the keys'
};
hipError_t launch_attention_forward(const AttentionCall& a, bool bf16, hipStream_t s);
hipError_t launch_attention_backward(const AttentionCall& a, bool bf16, hipStream_t s);

}  // namespace rbmoe
