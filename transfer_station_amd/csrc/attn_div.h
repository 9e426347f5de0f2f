/* attn_div.h -- division by what a call fixes, shared by the kernels and the host layer. */
#ifndef ATTN_DIV_H
#define ATTN_DIV_H

#include <stdint.h>

#include "attn_paged_rule.h"

/* n / d for 0 <= n < 2^31 by a product: mul = ceil(2^(31 + l) / d), l = ceil(log2 d), which is below 2^32 and off by
 * less than 2^l, so that the quotient is off by less than n 2^l / (d 2^(31 + l)) < 1 / d. Of the compiler's divisions, five
 * take a microsecond before a kernel's first load. */
struct attn_div {
    uint32_t mul, shift;
};
ATTN_HD struct attn_div attn_div_of(int d) {
    struct attn_div x = {0, 31};
    while ((int64_t)1 << (x.shift - 31) < d)
        ++x.shift;
    x.mul = (uint32_t)((((uint64_t)1 << x.shift) + (uint64_t)d - 1) / (uint64_t)d);
    return x;
}
ATTN_HD int attn_div_by(int n, struct attn_div x) { return (int)(((uint64_t)(uint32_t)n * x.mul) >> x.shift); }

#endif
