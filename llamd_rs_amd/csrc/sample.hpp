// sample.hpp -- arguments of the sampling kernels (sampling.hip) and their launcher. The entry point (sample.cpp) checks what the
// host can see; rules, random numbers and logits may hold anything.
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace llamd {

constexpr int SAMPLE_MOST = 1 << 20;  // logits of a row: their weights' sum stays inside 64 bits

// llamd_hip_sampling
struct __attribute__((aligned(16))) SampleRule {
    float temperature;
    int top_k;
    float top_p, min_p;
};

struct SampleArgs {
    const float *logits;  // [rows][ld]
    const SampleRule *how;
    const double *u;
    int32_t *ids;
    float *prob;  // may be null
    int ld, n;
};

int launch_sample(const SampleArgs &a, int rows, hipStream_t st);

}  // namespace llamd
