// Launches of kv_cache_kernels.hip.
#pragma once

#include <hip/hip_runtime.h>

#include <stddef.h>
#include <stdint.h>

#include "../../include/rbmoe.h"
#include "rbmoe_device.h"

namespace rbmoe {

// A pool of pages of `page_rows` rows.  Each page has one block a kv head:
//   keys    [page_rows][width]        width: head_dim rounded up to 64 or 128, zeros behind head_dim
//   values  [page_rows / g][width][g] g = the elements of 16 bytes: a lane of the decode kernel loads g keys of one column
//   scales  [2][page_rows] f32        (int8) of the keys, then of the values
struct CachePool {
    unsigned char* base;
    int pages, page_shift, kv_heads, head_dim, dtype;  // dtype: RBMOE_F32, RBMOE_BF16 or RBMOE_I8
    __host__ __device__ int width() const { return head_dim <= 64 ? 64 : 128; }
    __host__ __device__ int element() const { return dtype == RBMOE_F32 ? 4 : dtype == RBMOE_BF16 ? 2 : 1; }
    __host__ __device__ size_t half_bytes() const { return ((size_t)width() * element()) << page_shift; }
    __host__ __device__ size_t block_bytes() const { return 2 * half_bytes() + (dtype == RBMOE_I8 ? (size_t)8 << page_shift : 0); }
};
size_t cache_bytes(const CachePool& p);

struct CacheRows {
    CachePool pool;
    void* k;  // [rows, kv_heads, head_dim], rows *_stride elements apart
    void* v;
    long long k_stride, v_stride;
    const int64_t* slots;
    int rows;
};
hipError_t launch_cache_write(const CacheRows& a, bool bf16_rows, hipStream_t s);
hipError_t launch_cache_read(const CacheRows& a, bool bf16_rows, hipStream_t s);

struct DecodeCall {
    CachePool pool;
    const void* q;  // [sequences, heads, head_dim]
    void* out;      // the same without gaps
    long long q_stride;
    const int32_t* tables;  // [sequences][table_stride]
    const int32_t* lengths;
    int sequences, heads, table_pages, longest;
    int ranges;  // decode_plan's
    bool many;
    float scale;
    float* partial;     // [ranges + sequences][heads][width]: part range + sequence
    float* statistics;  // [ranges + sequences][heads][2]: reference of the exponents, sum
};
// ranges > 0: the tiles of all sequences in so many equal ranges; 0: a workgroup a sequence, `many`: of many waves.
struct DecodePlan {
    int ranges;
    bool many;
};
DecodePlan decode_plan(int sequences, int kv_heads, int group, int longest);
size_t decode_partials(int sequences, int kv_heads, int group);  // parts of heads at most, for up to so many sequences
hipError_t launch_decode_attention(const DecodeCall& a, bool bf16_rows, hipStream_t s);

}  // namespace rbmoe
