// Launches of muon_kernels.hip.
#pragma once

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <stddef.h>
#include <stdint.h>

#include "rbmoe_device.h"

namespace rbmoe {

// A stack of matrices [count][rows][cols]: element (i, r, c) at p[i * stride + r * pitch + c].
struct MuonStack {
    const void* p = nullptr;
    size_t stride = 0;
    int pitch = 0;
};

constexpr int kMostMuonSide = 1 << 14;  // rows or columns: an operand's offsets are 32-bit
constexpr int kMostMuonSteps = 64;

struct MuonCall {
    int count = 0, rows = 0, cols = 0;
    int steps = 5;
    bool grad_bf16 = false;
    MuonStack grad;            // f32 or bf16
    // an update: momentum (f32, read and written) and weight (f32, read and written).  Otherwise `out` takes the result.
    MuonStack momentum, weight;
    float mu = 0.0f, keep = 1.0f, rate = 0.0f;  // weight <- keep * weight - rate * O
    bool nesterov = true;
    bool out_bf16 = false;
    MuonStack out;
    void* workspace = nullptr;
};

// What is wrong with a step's settings, or null.
inline const char* muon_settings_problem(float lr, float momentum, float decay, float scale, int steps) {
    if (!std::isfinite(lr)) return "the learning rate must be finite";
    if (!(momentum >= 0.0f && momentum < 1.0f)) return "the momentum must be in [0, 1)";
    if (!std::isfinite(decay) || decay < 0.0f) return "the weight decay must be finite and not negative";
    if (!std::isfinite(scale) || scale < 0.0f) return "the update's scale must be finite and not negative";
    if (steps < 1 || steps > kMostMuonSteps) return "the number of steps must be between 1 and 64";
    return nullptr;
}
// 0 stands for sqrt(max(1, rows / cols)): an update moves every output of a layer by about the same, whatever its width.
inline float muon_scale(float given, int rows, int cols) {
    return given > 0.0f ? given : std::sqrt(std::max(1.0f, (float)rows / (float)cols));
}

// The kernel that takes a product (0: A, 1: B, 2: X) of a call.
enum class MuonTile { Split32, Split64, Rows64, Rows128 };
MuonTile muon_tile(int count, int rows, int cols, int product);

size_t muon_workspace_bytes(int count, int rows, int cols);
hipError_t launch_muon(const MuonCall& c, hipStream_t s);

}  // namespace rbmoe
