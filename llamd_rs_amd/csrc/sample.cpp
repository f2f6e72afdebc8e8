// sample.cpp -- the C entry point of the sampling kernels (include/llamd_hip.h): argument checks.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/llamd_hip.h"
#include "errors.hpp"
#include "launch.hpp"
#include "sample.hpp"

using namespace llamd;

namespace {

bool overlap(const void *a, size_t na, const void *b, size_t nb) {
    const uintptr_t x = (uintptr_t)a, y = (uintptr_t)b;
    return a && b && x < y + nb && y < x + na;
}

}  // namespace

extern "C" int llamd_hip_sample(const float *logits, int ld, int n, int n_seq, const llamd_hip_sampling *how,
                                const double *u, int32_t *ids, float *prob) {
    static_assert(sizeof(llamd_hip_sampling) == sizeof(SampleRule), "a rule as the kernels read it");
    if (n <= 0 || n > SAMPLE_MOST || ld < n) return set_error("sample: n %d (1 to %d), rows %d apart", n, SAMPLE_MOST, ld);
    if (n_seq < 0 || n_seq > 65535) return set_error("sample: %d sequences (65535 at most)", n_seq);
    if (!n_seq) return 0;
    if (!logits || !how || !u || !ids) return set_error("sample: null logits, rules, random numbers or ids");
    if ((((uintptr_t)logits | (uintptr_t)ids | (uintptr_t)prob) & 3) || ((uintptr_t)how & 15) || ((uintptr_t)u & 7))
        return set_error("sample: rules must be 16-byte aligned, random numbers 8, the others 4");
    const size_t rows = n_seq, in = ((rows - 1) * ld + n) * 4;
    const void *out[2] = {ids, prob};
    for (const void *x : out)
        if (overlap(x, rows * 4, logits, in) || overlap(x, rows * 4, how, rows * 16) || overlap(x, rows * 4, u, rows * 8))
            return set_error("sample: ids or probabilities overlap what the call reads");
    if (overlap(ids, rows * 4, prob, rows * 4)) return set_error("sample: ids overlap the probabilities");
    SampleArgs a{};
    a.logits = logits;
    a.how = (const SampleRule *)how;
    a.u = u;
    a.ids = ids;
    a.prob = prob;
    a.ld = ld;
    a.n = n;
    return launch_sample(a, n_seq, lib_stream()) ? set_error("sample: launch") : 0;
}
