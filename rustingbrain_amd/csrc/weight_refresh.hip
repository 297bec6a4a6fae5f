// After an update on the device: the layer's stored weights, and the transposed copies of the backward products, from f32 matrices.
// What rbmoe_set_weight does on the host for one matrix, for a stack of them in one launch: bound by memory, every element read once
// and written once a copy.
#include "rbmoe_kernels.h"

namespace rbmoe {

namespace {

// Where element (row, col) of a matrix of `cols` columns lies: plain rows, or the matrix cores' operand order (pack_weight_bf16).
__device__ __forceinline__ size_t packed_at(int row, int col, int cols) {
    return ((size_t)(row >> 5) * (cols >> 4) + (col >> 4)) * 512 + ((row & 31) + 32 * ((col >> 3) & 1)) * 8 + (col & 7);
}

// A workgroup takes 32 x 32 of a matrix, through LDS for the transposed copy.  Elements beyond the matrix's own rows and columns (rounded
// expert widths) are zero.
template <typename WT, bool PACKED>
__global__ __launch_bounds__(256) void weight_refresh_kernel(WeightRefresh a) {
    __shared__ float tile[32][33];
    const int i = blockIdx.z, r0 = blockIdx.y * 32, c0 = blockIdx.x * 32, tid = threadIdx.x;
    const float* const src = a.src + (size_t)i * a.src_stride;
    WT* const dst = static_cast<WT*>(a.dst) + (size_t)i * a.dst_rows * a.dst_cols;
    // gate and up share one transposed matrix, side by side
    WT* const turned = static_cast<WT*>(a.turned) + (size_t)(i / a.side) * a.dst_cols * a.turned_cols;
    const int turned_col = (i % a.side) * a.dst_rows;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const int r = k * 8 + tid / 32, c = tid % 32;
        tile[r][c] = r0 + r < a.rows && c0 + c < a.cols ? src[(size_t)(r0 + r) * a.src_pitch + c0 + c] : 0.0f;
    }
    __syncthreads();
    if constexpr (PACKED) {  // (whole tiles: the widths are multiples of 64)
        const int lane = tid & 63, step = (tid >> 6) & 1;
        const int row = lane & 31, col = 16 * step + 8 * (lane >> 5);
        const bool turn = tid >= 128;
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = turn ? tile[col + e][row] : tile[row][col + e];
        WT* const to = turn ? turned + packed_at(c0 + row, turned_col + r0 + col, a.turned_cols) : dst + packed_at(r0 + row, c0 + col, a.dst_cols);
        Vec16<bf16_t>::store(reinterpret_cast<bf16_t*>(to), v);
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int y = k * 8 + tid / 32, x = tid % 32;
            if (a.write_dst && r0 + y < a.dst_rows && c0 + x < a.dst_cols)
                dst[(size_t)(r0 + y) * a.dst_cols + c0 + x] = from_f32<WT>(tile[y][x]);
            if (c0 + y < a.dst_cols && r0 + x < a.dst_rows)
                turned[(size_t)(c0 + y) * a.turned_cols + turned_col + r0 + x] = from_f32<WT>(tile[x][y]);
        }
    }
}

}  // namespace

hipError_t launch_weight_refresh(const WeightRefresh& a, bool bf16, bool packed, hipStream_t s) {
    const dim3 grid((a.dst_cols + 31) / 32, (a.dst_rows + 31) / 32, a.count);
    if (packed) {
        if (!bf16 || a.dst_cols % 32 != 0 || a.dst_rows % 32 != 0) return hipErrorInvalidValue;
        hipLaunchKernelGGL((weight_refresh_kernel<bf16_t, true>), grid, dim3(256), 0, s, a);
    } else if (bf16) {
        hipLaunchKernelGGL((weight_refresh_kernel<bf16_t, false>), grid, dim3(256), 0, s, a);
    } else {
        hipLaunchKernelGGL((weight_refresh_kernel<float, false>), grid, dim3(256), 0, s, a);
    }
    return hipGetLastError();
}

}  // namespace rbmoe
