// attn_launch.h -- host helpers of the launchers: template flags, plan recording, the device's size.
// Included by attn_kernels.hip.
#ifndef ATTN_LAUNCH_H
#define ATTN_LAUNCH_H

#include <hip/hip_runtime.h>
#include <stdarg.h>
#include <stdio.h>
#include <string.h>

#include <type_traits>

namespace {

// Calls f(std::integral_constant<bool, b>{}): turns a runtime flag into a template argument.
template <typename F> hipError_t with_flag(bool b, F &&f) {
    return b ? f(std::true_type{}) : f(std::false_type{});
}

// Plan recording (attn_flash_plan): while t_plan is set on the calling thread, each launch
// site writes one line per kernel it would launch ("name<template arguments> grid=x[,y,z]
// block=n", then the site's notes) into the caller's buffer instead of launching.
struct plan_buf {
    char *buf;
    size_t len, pos;
    bool truncated;
};
thread_local plan_buf *t_plan = nullptr;
const char *tf(bool b) { return b ? "true" : "false"; }

__attribute__((format(printf, 3, 4))) void plan_note(dim3 g, dim3 b, const char *fmt, ...) {
    plan_buf *p = t_plan;
    char line[256];
    va_list ap;
    va_start(ap, fmt);
    int n = vsnprintf(line, sizeof line, fmt, ap);
    va_end(ap);
    if (n < 0)
        n = 0;
    size_t used = (size_t)n < sizeof line ? (size_t)n : sizeof line - 1;
    int m = (g.y > 1 || g.z > 1)
                ? snprintf(line + used, sizeof line - used, " grid=%u,%u,%u block=%u\n", g.x, g.y,
                           g.z, b.x * b.y * b.z)
                : snprintf(line + used, sizeof line - used, " grid=%u block=%u\n", g.x,
                           b.x * b.y * b.z);
    used += (m > 0 && (size_t)m < sizeof line - used) ? (size_t)m : 0;
    if (p->pos + used + 1 > p->len) {
        p->truncated = true;
        return;
    }
    memcpy(p->buf + p->pos, line, used);
    p->pos += used;
    p->buf[p->pos] = '\0';
}

// Compute units of the current device (cached per device).
static int device_cus() {
    static int cus[64];
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64)
        return 256;
    if (cus[dev] <= 0) {
        int n = 0;
        if (hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess ||
            n <= 0)
            n = 256;
        cus[dev] = n;
    }
    return cus[dev];
}
} // namespace

#endif
