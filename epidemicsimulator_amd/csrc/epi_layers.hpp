// Layer operators of the engine: dropout from a counter-based generator and layer normalisation, forward and
// backward, on device memory.  The launchers below are shared by the C entry points (epi_layers.hip) and by the
// learners (epi_agents.hip), which run them between the linear layers of their networks.
#pragma once
#include <hip/hip_runtime.h>

#include <cstddef>
#include <cstdint>

namespace epi {

// Dropout as the kernels need it.  Philox4x32-10 (Salmon, Moraes, Dror and Shaw, "Parallel random numbers: as easy
// as 1, 2, 3", 2011) with key = seed and counter = (column / 8, row, offset) gives four words = eight draws of 16 bits,
// one for each of eight consecutive columns; a unit is dropped when its draw is below `threshold` = p in units of
// 2^-16, and a kept one is multiplied by 65536 / (65536 - threshold), which makes the mean exact for the rounded p.
struct DropArgs {
    uint32_t threshold;          // 0: no dropout; 65536: every unit is dropped
    double scale;
    uint32_t key[2], offset[2];
    const int64_t* offset_dev;   // added to offset when not NULL: a captured graph draws anew on every replay
};
DropArgs make_drop(double p, int64_t seed, int64_t offset, const int64_t* offset_dev);

// Weights of several networks in one call, of doubles (one set of rows each): rows k * set_rows .. + set_used[k] - 1 belong to
// set k and use weight / bias number set_index[k]; the rows behind set_used[k] are neither read nor written.
// set_ctr[2 k .. 2 k + 1] replaces the dropout offset of set k, and its rows count from zero.
struct NormSets {
    int count, set_rows;
    const int32_t *set_used, *set_index;
    const uint32_t* set_ctr;
    int64_t weight_stride;       // elements from one set's weights to the next one's
};

struct NormArgs {
    int64_t rows, cols, x_stride, y_stride, dy_stride;   // y_stride: of y (forward) or dx (backward)
    const void *x, *dy, *weight, *bias;                  // weight and bias may be NULL: ones and zeros
    void *y, *dx;
    void *mean, *rstd;           // [rows], double for doubles, else float
    void *dweight, *dbias;       // [cols], or [sets][cols] with sets
    void* workspace;
    double eps;
    double inv_cols;             // 1 / cols, set by the launchers
    DropArgs drop;
    NormSets sets;               // sets.count == 0: one set of weights
};

enum LayerType { kF64 = 0, kF32 = 1, kBF16 = 2, kF16 = 3 };

hipError_t launch_dropout(LayerType type, int64_t rows, int64_t cols, int64_t x_stride, int64_t y_stride, const void* x,
                          void* y, const DropArgs& drop, hipStream_t s);
hipError_t launch_norm_forward(LayerType type, const NormArgs& a, hipStream_t s);
size_t norm_backward_workspace(LayerType type, int64_t rows, int64_t cols, bool drop);
hipError_t launch_norm_backward(LayerType type, const NormArgs& a, hipStream_t s);

}  // namespace epi
