// nl_ops.h -- what nl_ops.hip has for the layer-stack models' host (nl_stack.hip): launches of the feed-forward of experts.
#pragma once
#include "../../include/nanollama_ops.h"

#include <hip/hip_runtime.h>

namespace nl {

void set_error(const char *message);      // what nl_last_error(NULL) returns on this thread (nl_stack.hip)

struct RouteParams {
    const float *logits, *bias;           // [n][ld]; [experts] or null
    long long ld;
    int n, experts, k, sigmoid, renorm;
    float scale;
    int *ids;                             // [n][k]
    float *weights;
};
hipError_t launch_route(const RouteParams &P, hipStream_t st);

struct ExpertsParams {
    const void *x, *gate, *up, *down;     // [n][ldx]; [experts][ff][dim] twice; [experts][dim][ff]
    long long ldx;
    const int *ids;                       // [n][k]
    const float *weights;
    int n, k, experts, dim, ff, act;      // act: NL_ACT_*
    // workspace (experts_layout)
    int *offs, *order;                    // first place of every expert [experts + 1]; place -> slot (token * k + j)
    void *h;                              // [place][ff] activations in the element type, or [slot][ff] in 32 bits
    void *h_rest;                         // [place][ff] what their rounding left, in the element type, or null; launch_experts has it
    float *part;                          // [slot][dim] weighted results
    // launch_experts has these: where the sums of a few tokens go at once, if anywhere
    void *y;
    const float *res, *add;
    float *res_out;
    long long ldy, ldres, ldadd, ldo;
    float scale;
};
// bytes of the workspace and where its parts start
struct ExpertsLayout { size_t offs, order, h, part, bytes; };
ExpertsLayout experts_layout(int n, int k, int experts, int dim, int ff, int dtype);
void place_experts(ExpertsParams &P, void *workspace, const ExpertsLayout &L);

// the sum of a token's results (part, ids; null: none) and of `base` (null: none) is d:  x_out = x + add + scale gate v, h = norm(x_out) pre
struct CloseParams {
    const float *x, *add, *base;          // add: a second addend or null
    long long ldx, ldadd, ldbase;
    const void *d;                        // rows of the element type, instead of part and base
    long long ldd;
    const float *part;                    // [slot][dim]
    const int *ids;                       // null: a row of part a token
    int k, experts;
    const float *post, *gate, *pre;
    long long ldgate;
    float *x_out;                         // null: the sum goes to y, in the element type
    long long ldxo;
    void *h, *y;
    long long ldh, ldy;
    int n, dim;
    float eps, scale;
};
hipError_t launch_close(const CloseParams &P, int dtype, hipStream_t st);
// the experts' products of P's tokens and the close C of their sums (its part, ids, k, experts, n and dim are filled in, base and d stay null)
hipError_t launch_experts(const ExpertsParams &P, const CloseParams &C, int dtype, hipStream_t st);

}  // namespace nl
