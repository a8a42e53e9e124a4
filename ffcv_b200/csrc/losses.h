// What the losses share (cross_entropy.cu, linear_cross_entropy.cu, distillation.cu).
#pragma once

#include "training.h"
#include "two.h"

namespace ffcvb {

// (*loss = sum or mean of rows' losses, always added in the same order; `counted` rows, or all where it is NULL.)
void launch_mean(const float *row_loss, int64_t rows, const float *counted, bool mean, float *loss, cudaStream_t stream);
// (*counted = rows whose label is not `ignore`.)
void launch_count(const void *labels, int64_t rows, int64_t stride, int64_t ignore, float *counted, cudaStream_t stream);

#ifdef __CUDACC__

// (Differences are taken before the factor: a row masked with the type's lowest value has no product with it.)
constexpr float kLog2e = 1.4426950408889634f;
__device__ __forceinline__ float exp2_of(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float exp_of(float x) { return exp2_of(x * kLog2e); }

// What a row's target is besides probabilities per class: at most two classes with their weights, and the same
// `flat` for all.
struct Picks {
    long long label[2];
    float weight[2];
    float flat;
    float total;  // S
    bool ignored, bad;
};

template <typename Args> __device__ __forceinline__ Picks picks_of(const Args &a, long long row) {
    Picks p{{-1, -1}, {0.0f, 0.0f}, a.smoothing / (float)a.classes, 0.0f, false, false};
    const float sure = 1.0f - a.smoothing;
    if (a.target_kind == FFCVB_TARGET_LABELS) {
        p.label[0] = static_cast<const int64_t *>(a.target)[row * a.target_stride];
        p.weight[0] = sure;
        p.ignored = a.has_ignore && p.label[0] == a.ignore_index;
        p.bad = p.label[0] < 0 || p.label[0] >= a.classes;
        p.total = sure + a.smoothing;
    } else if (a.target_kind == FFCVB_TARGET_MIXED) {
        const float *m = static_cast<const float *>(a.target) + row * a.target_stride;
        const float l0 = m[0], l1 = m[1], lam = m[2];
        p.bad = !(l0 >= 0.0f && l0 < (float)a.classes && l1 >= 0.0f && l1 < (float)a.classes);
        if (!p.bad) {
            p.label[0] = (long long)l0;
            p.label[1] = (long long)l1;
        }
        p.weight[0] = sure * lam;
        p.weight[1] = sure * (1.0f - lam);
        p.total = p.weight[0] + p.weight[1] + a.smoothing;
    }
    return p;
}

__device__ __forceinline__ void copy16(uint32_t to, const void *from) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
}

constexpr float kLowest = -3.402823466e38f;

#endif

} // namespace ffcvb
