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
    float* parts;  // [shares][key_rows, kv_heads][2][head_dim]: sums of dk and dv over a share of a group's heads
    int part_rows; // room for so many rows of a share
    int shares;    // set by the launch
};
// rows of f32 sums [2][head_dim], for every head of a group, that the backward pass of up to so many rows may share out
int attention_part_rows(int backward_rows, int kv_heads, int group);
hipError_t launch_attention_forward(const AttentionCall& a, bool bf16, hipStream_t s);
hipError_t launch_attention_backward(const AttentionCall& a, bool bf16, hipStream_t s);

}  // namespace rbmoe
