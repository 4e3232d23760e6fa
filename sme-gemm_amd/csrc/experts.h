// Launch interface of expert routing (route.hip) and the experts' products
// (experts.hip). Internal to the library.
#pragma once

#include "fp8.h"

namespace smg {

enum LogitType : int { LOGIT_F32 = 0, LOGIT_F16 = 1, LOGIT_BF16 = 2 };
constexpr uint32_t ROUTE_MAX_EXPERTS = 1024, ROUTE_MAX_TOP = 64, ROUTE_MAX_GROUPS = 64;

struct RouteArgs {
    const void *logits;   // [rows][experts]
    const float *bias;    // [experts] or null
    int32_t *ids;         // [rows][top_k]
    float *weights;       // [rows][top_k]
    uint32_t rows, experts, top_k;
    uint32_t sigmoid;     // else softmax
    uint32_t groups, top_groups;
    uint32_t renormalize;
    float scale;
};
hipError_t launch_route(const RouteArgs &a, int logit_type, hipStream_t s);

// The experts of a mixture: gate and up (n = hidden width, k = model width) and down
// (n = model width, k = hidden width), all of one count.
struct ExpertSet {
    Fp8Mat gate, up, down;
    uint32_t act;  // EP_ACT_SILU or EP_ACT_GELU
};

// A tile slot: its expert, whose tiles are `count` from number `first` on, of 256 rows each
// but for the last if `half` (128), and whose row tiles of 16 are rt .. rt_end - 1.
struct ExpertTile {
    uint32_t expert, half, first, count, rt, rt_end;
};
// Where the assignments (row r's j-th expert, number r * top_k + j) of a call go: one
// expert's after another, each expert's rows padded to a multiple of 64, in device
// memory written by launch_expert_plan.
struct ExpertPlan {
    uint32_t *head;       // EXPERT_TILES: tiles; EXPERT_ROWS: padded rows
    ExpertTile *tiles;    // [max_tiles]
    int32_t *place;       // [assignments] the padded row, -1: no expert
    int32_t *rank;        // [assignments] the place among its expert's rows, -1
    int32_t *source;      // [max_rows] the assignment, -1: padding
    uint32_t assignments, top_k, experts;
    uint32_t max_rows, max_tiles;  // what any choice of experts may need
};
enum : uint32_t { EXPERT_TILES = 0, EXPERT_ROWS = 1 };

// The plan's rows times their expert's weights: with `up` the hidden values act(a W) *
// (a up), quantized into h, else C to dst [max_rows][w.n]. exact (with `up`): sums that lose
// nothing but f32's roundings, at the rate of f16.
hipError_t launch_fp8_grouped(const Fp8Mat &w, const Fp8Mat *up, uint32_t act, const ExpertPlan &p, Fp8Rows a, Fp8Rows h,
                              float *dst, bool exact, hipStream_t s);

// out [rows][d] (16-bit, of x's type), or y (f32) += out: the weighted sum over each
// row's experts. ids outside 0 .. experts - 1 stand for no expert.
struct ExpertCall {
    const uint16_t *x;       // [rows][d]
    const int32_t *ids;      // [rows][top_k]
    const float *weights;    // [rows][top_k]
    uint16_t *out;           // or null
    float *y;                // or null
    uint32_t rows, top_k;
    bool bf16;
};
size_t experts_scratch_bytes(const ExpertSet &e, const ExpertCall &c);
size_t experts_scratch_bytes(const ExpertSet &e, size_t rows, size_t top_k);  // the most, x at any address
hipError_t launch_experts(const ExpertSet &e, const ExpertCall &c, void *scratch, hipStream_t s);

}  // namespace smg
