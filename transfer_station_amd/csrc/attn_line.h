// attn_line.h -- the decode line (attn_quota in attn_paged_rule.h) as a wave of the decode kernels sees it, and the wave's
// sums and maxima that it takes. For arguments A with B, teams and nsplit, and U with at(a, i) (the units of sequence i, 0
// past the last), one(a) (those of the only one) and heads(a) (how often the line is walked).
#ifndef ATTN_LINE_H
#define ATTN_LINE_H

#include "attn_device.h"
#include "attn_paged_rule.h"

namespace {

// Sum or maximum over the wave, in every lane.
template <bool MAX> __device__ __forceinline__ int wave_all(int x) {
    auto op = [](int p, int q) { return MAX ? max(p, q) : p + q; };
    x = op(x, __builtin_amdgcn_update_dpp(x, x, 0x128, 0xf, 0xf, false)); // row_ror:8, 4, 2, 1
    x = op(x, __builtin_amdgcn_update_dpp(x, x, 0x124, 0xf, 0xf, false));
    x = op(x, __builtin_amdgcn_update_dpp(x, x, 0x122, 0xf, 0xf, false));
    x = op(x, __builtin_amdgcn_update_dpp(x, x, 0x121, 0xf, 0xf, false));
    const auto p = __builtin_amdgcn_permlane16_swap((unsigned)x, (unsigned)x, false, false);
    x = op((int)p[0], (int)p[1]);
    const auto r = __builtin_amdgcn_permlane32_swap((unsigned)x, (unsigned)x, false, false);
    return op((int)r[0], (int)r[1]);
}

// x plus those of the lanes below (DPP row shifts, then the rows' last lanes broadcast to the rows behind).
__device__ __forceinline__ int wave_scan(int x) {
    x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, true); // row_shr:1, 2, 4, 8
    x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, true);
    x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, true);
    x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, true);
    x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false); // row_bcast:15 into rows 1 and 3
    return x + __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false); // row_bcast:31 into rows 2 and 3
}

// The decode line (attn_quota) as a wave sees it, 64 sequences at a time: a kv head's units and the quota.
// One sequence needs no sum, and up to 64 are read once.
struct line {
    int total, quota;
    int n, sum; // of sequence `lane`: units, and units up to and with it
};
template <typename U, typename A> __device__ __forceinline__ line line_at(const A &a, int lane) {
    line l;
    int most;
    if (a.B == 1) {
        l.n = l.sum = l.total = most = U::one(a);
    } else {
        l.n = U::at(a, lane);
        l.sum = wave_scan(l.n);
        l.total = __builtin_amdgcn_readlane(l.sum, 63);
        int m = l.n;
        for (int i0 = 64; i0 < a.B; i0 += 64) {
            const int n = U::at(a, i0 + lane);
            m = max(m, n);
            l.total += __builtin_amdgcn_readlane(wave_scan(n), 63);
        }
        most = uniform(wave_all<true>(m));
    }
    l.quota = uniform(attn_quota(l.total, most, U::heads(a), a.teams, a.nsplit));
    return l;
}
// The sequence that unit `at` of a kv head's line belongs to, and the units before that.
template <typename U, typename A>
__device__ __forceinline__ int seq_of_unit(const A &a, const line &l, int lane, int at, int &before) {
    before = 0;
    if (a.B == 1)
        return 0;
    int n = l.n, sum = l.sum, base = 0;
    for (int i0 = 0;;) {
        const uint64_t past = __builtin_amdgcn_ballot_w64(base + sum > at);
        if (past != 0) {
            const int k = __builtin_ctzll(past);
            before = base + __builtin_amdgcn_readlane(sum - n, k);
            return i0 + k;
        }
        base += __builtin_amdgcn_readlane(sum, 63);
        i0 += 64;
        if (i0 >= a.B) // not reached for a unit of the line
            return 0;
        n = U::at(a, i0 + lane);
        sum = wave_scan(n);
    }
}

// The units of a line before sequence b.
template <typename U, typename A>
__device__ __forceinline__ int units_before(const A &a, const line &l, int lane, int b) {
    if (a.B == 1)
        return 0;
    int n = l.n, sum = l.sum, base = 0;
    for (int i0 = 0; i0 + 64 <= b; n = U::at(a, i0 + lane), sum = wave_scan(n)) {
        base += __builtin_amdgcn_readlane(sum, 63);
        i0 += 64;
    }
    return base + __builtin_amdgcn_readlane(sum - n, b & 63);
}

} // namespace

#endif
