// groupnorm.h -- group norm with an activation over channels-last data: what
// the C ABI (ops.cpp) hands to the kernels (groupnorm.hip).
//
//   y = (x - mean) / sqrt(var + eps) * weight_c + bias_c,  then act(y), or
//   y * act(gate);  mean and var over `rows` rows and channels / groups channels
#pragma once

#include <hip/hip_runtime.h>

#include "ssla_hip.h"

namespace ssla {

enum GroupNormKind { kGroupLanes, kGroupOnePass, kGroupTwoPass };

struct GroupNormArgs {
    const void *x, *gate, *weight, *bias;
    void* out;
    long long xn, xr, gn, gr, on, orow;   // strides, elements: item, row
    double* ws;                           // [item][part][group] sum, sum of squares
    int n, rows, channels, groups, act;
    float eps;
    // how the call is cut (group_norm_plan)
    int vec;                              // channels of a piece: 16 bytes where alignment allows
    int kind;                             // kGroupLanes, kGroupOnePass, kGroupTwoPass
    int threads, reps;                    // of a workgroup; pieces a thread keeps (one pass).  Lanes:
                                          // pieces a lane keeps; lanes of a group (over 64: a workgroup)
    int gb, blocks, np;                   // groups of a workgroup; workgroups along the groups; pieces of
                                          // a workgroup's row
    int parts;                            // workgroups along the rows; 0: not two passes
    double inv_count;                     // 1 / values of a group
};

void group_norm_plan(GroupNormArgs& a, int dtype);
hipError_t group_norm_launch(const GroupNormArgs& a, int dtype, hipStream_t st);

}  // namespace ssla
