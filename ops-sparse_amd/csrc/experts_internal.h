// Launcher interface between the host checks of the experts' operators
// (experts_host.cpp) and their gfx950 kernels.  Nothing here is public.
#pragma once

#include <cstddef>
#include <cstdint>

#include "cann_ops_sparse.h"

namespace aclsp {

// The most experts a router's row may have (64 for each of 16 lanes) and the
// most of them a token may choose (one per lane of a wave).
constexpr int64_t kMaxRouteExperts = 1024;
constexpr int64_t kMaxRouteK = 64;
// The longest contraction of 8-bit products whose sum cannot leave 32 bits:
// 2^14 * 131071 < 2^31.
constexpr int64_t kMaxScaledK = 131071;

// What a launcher returns when a grid would not fit.  Its workgroups are
// numbered in 31 bits, and along a dimension it has fewer than 2^32 threads: a
// larger one is launched without an error, with its size cut to 32 bits.
constexpr int kTooLarge = 1;
inline bool GridFits(int64_t blocks, int64_t threads)
{
    return blocks <= INT32_MAX && blocks * threads <= UINT32_MAX;
}

struct RouteLaunch {
    int64_t tokens, experts, k;
    const void* logits;  // null: the choice is given in ids
    int64_t ld;
    aclDataType type;
    int32_t normalize;
    float* weights;
    int32_t* ids;  // read when logits is null
    int32_t* offsets;
    int32_t* row_tokens;
    int32_t* places;
    int32_t* hist;  // the caller's buffer: RouteBlocks * experts counts
};

// Workgroups of the routing kernels, and so rows of their histogram.
int64_t RouteBlocks(int64_t tokens);
int LaunchRoute(const RouteLaunch& l, void* stream);

struct RouteGradLaunch {
    int64_t tokens, experts, k;
    const void* logits;
    int64_t ld;
    aclDataType type;
    int32_t normalize;
    const float* weights;
    const int32_t* ids;
    const float* grad_weights;
    void* grad_logits;
    int64_t ld_grad;
};
int LaunchRouteGrad(const RouteGradLaunch& l, void* stream);

struct CombineLaunch {
    int64_t tokens, k, width, rows;
    const int32_t* places;
    const float* weights;  // null: ones
    const void* y;
    int64_t ldy;
    aclDataType y_type;
    void* out;
    int64_t ldo;
    aclDataType out_type;
    int32_t* head;  // null: no lists for the gradient
    int32_t* next;
};
int LaunchCombine(const CombineLaunch& l, void* stream);

struct CombineGradLaunch {
    int64_t tokens, k, width, rows, groups;
    const int32_t* offsets;  // of the plan that the places are of; null: any places, with head and next
    const int32_t* places;
    const float* weights;  // null: ones
    const void* y;         // null: no gradient of the weights
    int64_t ldy;
    const void* grad_out;
    int64_t ldo;
    aclDataType type;
    void* grad_y;  // null: not wanted
    int64_t ld_grad_y;
    float* grad_weights;  // null: not wanted
    int32_t* head;  // the caller's buffer: one per row
    int32_t* next;  // and one per assignment
    bool listed;    // they hold the lists already
};
int LaunchCombineGrad(const CombineGradLaunch& l, void* stream);

struct GroupedLaunch {
    int64_t groups, rows, n, k;
    const int32_t* offsets;    // null: one group of all rows
    const int32_t* row_index;  // null: row r of C is row r of A
    int64_t rows_a;
    const void* a;
    int64_t lda;
    const void* b;
    int64_t ldb, stride_b;
    int32_t b_trans;  // B_g is [n, k] (1) or [k, n] (0)
    aclDataType ab_type;
    const float* scale_a;  // 8-bit products: one per row of A
    const float* scale_b;  // and one per group and column
    void* c;
    int64_t ldc;
    aclDataType c_type;
};
int LaunchGroupedMM(const GroupedLaunch& l, void* stream);

struct GroupedGradLaunch {
    int64_t groups, rows, n, k;
    const int32_t* offsets;
    const int32_t* row_index;
    int64_t rows_x;
    const void* grad;  // [rows, n]
    int64_t ldg;
    const void* x;  // [rows_x, k]
    int64_t ldx;
    aclDataType type;
    void* w;  // per group [n, k]
    int64_t ldw, stride_w;
    aclDataType w_type;
};
int LaunchGroupedMMGrad(const GroupedGradLaunch& l, void* stream);

}  // namespace aclsp
