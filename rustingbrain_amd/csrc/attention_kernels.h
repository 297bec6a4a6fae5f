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
    int sequences, query_rows, key_rows, longest_queries, longest_keys;  // (longest_*: as the call names them)
    int most_queries, most_keys;                                         // and what of them the arrays have room for: sizes of launches
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

// Which rows of a sequence there are, and how they stand to its keys: row r (of those that are there) sees the keys up to r + ahead.
struct Sequence {
    int q0, nq, k0, nk, ahead;
};
// Whatever the arrays of begins and counts hold: a sequence's rows and keys are those of its `count` from `begin` on that lie inside the arrays, and
// each sees what it would see if all were there.  (ahead is cut where nothing changes any more, so that sums of it and a row stay in range.)
__host__ __device__ inline Sequence cut_sequence(int query_begin, int query_count, int key_begin, int key_count, int query_rows, int key_rows,
                                                 int longest_queries, int longest_keys) {
    auto least = [](long long a, long long b) { return a < b ? a : b; };
    auto most = [](long long a, long long b) { return a < b ? b : a; };
    const long long nq = least(most(query_count, 0), longest_queries), nk = least(most(key_count, 0), longest_keys);
    Sequence s;
    s.q0 = (int)least(most(query_begin, 0), query_rows);
    s.k0 = (int)least(most(key_begin, 0), key_rows);
    s.nq = (int)most(least(query_begin + nq, query_rows) - s.q0, 0);
    s.nk = (int)most(least(key_begin + nk, key_rows) - s.k0, 0);
    const long long missing_queries = most(-(long long)query_begin, 0), missing_keys = most(-(long long)key_begin, 0);  // in front
    s.ahead = (int)most(least(nk - nq + missing_queries - missing_keys, s.nk - 1), -s.nq);
    return s;
}
// rows of f32 sums [2][head_dim], for every head of a group, that the backward pass of up to so many rows may share out
int attention_part_rows(int backward_rows, int kv_heads, int group);
hipError_t launch_attention_forward(const AttentionCall& a, bool bf16, hipStream_t s);
hipError_t launch_attention_backward(const AttentionCall& a, bool bf16, hipStream_t s);

}  // namespace rbmoe
