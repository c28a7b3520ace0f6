// deepipr_host.h -- internal (not installed): the host-side plumbing that deepipr_hip.hip shares with the translation units that
// hold C entry points of their own (deepipr_gradnorm.hip, deepipr_mx4.hip): error text, launch check, in-situ timing.
#ifndef DEEPIPR_HOST_H
#define DEEPIPR_HOST_H
#include <hip/hip_runtime.h>
#include <hip/hip_ext.h>

#include "../../include/deepipr_hip.h"
#include "deepipr_conv_plan.h"

// Sets the thread's error text and returns `code`.
DIPR_HIDDEN int dipr_fail(int code, const char *fmt, ...) __attribute__((format(printf, 2, 3)));
// DEEPIPR_OK, or DEEPIPR_ELAUNCH with the text of hipGetLastError().
DIPR_HIDDEN int dipr_check_launch(const char *what);

// One timed kernel: while deepipr_profile_enable is on, `a` / `b` are the dispatch's own start / stop events of the FIRST launch
// that goes through DIPR_LAUNCH with this scope; off (the normal case) both are null.
struct DIPR_HIDDEN DiprProf {
    explicit DiprProf(int kernel);
    ~DiprProf();
    DiprProf(const DiprProf &) = delete;
    int k;
    hipEvent_t a = nullptr, b = nullptr;
    bool used = false;
    double bytes = 0.0;                  // algorithmic bytes (FLOPs for the matrix product) of the timed launch
};

#define DIPR_LAUNCH(prof, kernel, grid, block, st, ...)                                                 \
    do {                                                                                                \
        if ((prof).a && !(prof).used) {                                                                 \
            (prof).used = true;                                                                         \
            hipExtLaunchKernelGGL(kernel, grid, block, 0, st, (prof).a, (prof).b, 0, __VA_ARGS__);      \
        } else {                                                                                        \
            hipLaunchKernelGGL(kernel, grid, block, 0, st, __VA_ARGS__);                                \
        }                                                                                               \
    } while (0)
#endif
