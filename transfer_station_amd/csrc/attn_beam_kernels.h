// attn_beam_kernels.h -- gfx950 kernels of beam search: the K best continuations of each batch entry's beams over the
// vocabulary (attn_beam_select), and the paged cache's sequences following their parents (attn_kv_reorder). Part of
// attn_kernels.hip.
#ifndef ATTN_BEAM_KERNELS_H
#define ATTN_BEAM_KERNELS_H

#include "attn_beam_rule.h"
#include "attn_flash.h"
#include "attn_device.h"
#include "attn_launch.h"

namespace {

// Floats and doubles as unsigned numbers of the same order, -0 as 0; 0 stands for none (a NaN with the sign bit).
__device__ __forceinline__ uint32_t ordered(float x) {
    const uint32_t u = __builtin_bit_cast(uint32_t, x + 0.f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float unordered(uint32_t u) {
    return __builtin_bit_cast(float, u & 0x80000000u ? u & 0x7fffffffu : ~u);
}
__device__ __forceinline__ uint64_t ordered(double x) {
    const uint64_t u = __builtin_bit_cast(uint64_t, x + 0.0);
    return u >> 63 ? ~u : u | 0x8000000000000000ull;
}
__device__ __forceinline__ double unordered(uint64_t u) {
    return __builtin_bit_cast(double, u >> 63 ? u & 0x7fffffffffffffffull : ~u);
}
constexpr float kLog2E = 1.44269504088896341f;
constexpr uint32_t kOrderedNegInf = 0x007fffffu; // ordered(-inf): what is above it is a candidate
// A test of the bits, which the compiler must not see as one of a float: those are compiled as if there were no NaN.
__device__ __forceinline__ bool finite(float x) {
    return (opaque(__builtin_bit_cast(uint32_t, x)) & 0x7f800000u) != 0x7f800000u;
}

// A value that at least K of the wave's 64 N numbers reach (`none` where fewer are above that), and hardly more: from a
// lane's largest up or down in growing steps until the count passes K, then by halves until it is between K and K + 7.
template <int N> __device__ __forceinline__ uint32_t wave_kth(const uint32_t (&x)[N], uint32_t none, uint32_t step, int K) {
    auto count = [&](uint32_t y) {
        int n = 0;
#pragma unroll
        for (int i = 0; i < N; ++i)
            n += (int)__builtin_popcountll(__builtin_amdgcn_ballot_w64(x[i] >= y));
        return n;
    };
    if (count(none + 1) < K)
        return none;
    uint32_t first = x[0];
#pragma unroll
    for (int i = 1; i < N; ++i)
        first = max(first, x[i]);
    uint32_t lo = max((uint32_t)__builtin_amdgcn_readfirstlane((int)first), none + 1), hi = lo; // count(lo) >= K > count(hi)
    if (count(lo) >= K) {
        do {
            lo = hi;
            if (hi > ~step) {
                hi = ~0u;
                break;
            }
            hi += step;
            step = max(step, step << 1);
        } while (count(hi) >= K);
    } else {
        do {
            hi = lo;
            if (lo <= none + step) {
                lo = none + 1;
                break;
            }
            lo -= step;
            step = max(step, step << 1);
        } while (count(lo) < K);
    }
    while (count(lo) >= K + 8 && lo + 1 < hi) {
        const uint32_t mid = lo + (hi - lo) / 2;
        if (count(mid) >= K)
            lo = mid;
        else
            hi = mid;
    }
    return lo;
}

// The threads' sum, in every thread. red: four ints; ends with a barrier, so that red may be used again.
__device__ __forceinline__ int wg_sum(int x, int *red, int tid) {
#pragma unroll
    for (int i = 1; i < 64; i <<= 1)
        x += __shfl_xor(x, i);
    if ((tid & 63) == 0)
        red[tid >> 6] = x;
    __syncthreads();
    x = red[0] + red[1] + red[2] + red[3];
    __syncthreads();
    return x;
}

// ------------------------------------------------------------------------------------------
// One chunk of a row: its largest logit m, the sum of exp(x - m), and its K largest logits, of equals those at the lowest
// index. x - m is taken first, for all sizes of x: m log2(e), rounded, is off by more than an exponent of 1 from 2^24 on,
// and has none at a mask of the type's lowest value.
// The four waves take neighbouring pieces of it, a step of 4 KB at a time with the next on its way, each lane with a
// maximum and sum of its own. A wave's threshold is a value that at least K of its lanes have reached (wave_kth; past K = 32, K of
// its lanes' halves: the least of 64 lanes is no threshold), taken anew as the number of steps doubles: some K logits pass it
// per doubling. They go to LDS; at the end those below the best
// of the four thresholds fall away, and each of the rest counts how many are ahead of it. Each logit is read once: 512 rows of
// 128256 in bf16, 131 MB, 32 us (4.1 TB/s where a copy reaches 4.9; eight instructions and an exponential, at a quarter of
// their rate, per logit and lane), four rows of 50257 in fp32 5.4.
// Where more pass in one wave than LDS has room for, the K-th element's value and index are searched for bit by bit, up to 66
// passes over the chunk in memory. That is so for equal and for ascending logits, for pieces of which nearly all have one finite
// value (64 entries of 8 beams over 128256 in bf16, all but 100 of a row at the lowest value: 5.7 ms, at -inf 32 us), and for
// large K over many steps, since what has passed stays to the end: of normal logits some K pass per doubling (16 entries of 64
// beams over 128256 in bf16, 16 steps to a wave: K = 24 67 us, K = 32 5.4 ms, K = 64 11.1; 4 of 64 in fp32, 8 steps: K = 40 44 us,
// K = 48 1.1 ms, K = 64 2.9). Among 1024 rows some wave is there with K = 64 from 4 steps on, 48 from 8, 32 from 16, 24 from 32.
// ------------------------------------------------------------------------------------------
constexpr int kBeamRoom = 256, kBeamBest = 512; // places for a wave's logits, and for those that are ranked

template <typename T> __global__ __launch_bounds__(256, 4) void attn_beam_chunk_kernel(const attn_beam_args a) {
    constexpr int VEC = 16 / sizeof(T), NV = 4, STEP = ATTN_BEAM_STEP(sizeof(T)); // logits of a wave's step
    static_assert(STEP == 64 * VEC * NV, "");
    __shared__ uint64_t room[4 * kBeamRoom], best[kBeamBest];
    __shared__ float redm[4], reds[4];
    __shared__ uint32_t redu[4];
    __shared__ int redi[4], redn[4], kept;
    const int row = wg_id_x() / a.chunks, chunk = wg_id_x() - row * a.chunks, tid = wi_id_x(), lane = tid & 63;
    const int w = uniform(tid >> 6);
    if ((a.done && a.done[row]) || !finite(a.scores[row]))
        return;
    const T *x = reinterpret_cast<const T *>(a.logits) + row * a.row;
    const int first = chunk * 4 * a.steps * STEP, begin = first + w * a.steps * STEP;
    const int end = min(begin + a.steps * STEP, a.V);
    if (tid == 0)
        kept = 0;
    auto value = [](u32x4 v, int i) {
        if constexpr (sizeof(T) == 2)
            return __builtin_bit_cast(float, i & 1 ? v[i >> 1] & 0xffff0000u : v[i >> 1] << 16);
        const uint32_t e = v[i]; // a value: of an element in place bit_cast takes the vector's first
        return __builtin_bit_cast(float, e);
    };
    auto bits_of = [](T t) -> uint32_t {
        if constexpr (sizeof(T) == 2)
            return t;
        else
            return __builtin_bit_cast(uint32_t, t);
    };
    // Vector j of the step at `at` is 64 VEC j + VEC lane on; past the row's end there are logits of -inf.
    auto load = [&](int at, u32x4 *v) __attribute__((always_inline)) {
        if (at + STEP <= a.V) {
#pragma unroll
            for (int j = 0; j < NV; ++j)
                v[j] = __builtin_nontemporal_load(reinterpret_cast<const u32x4_a2 *>(x + at + (64 * j + lane) * VEC));
        } else {
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const int k = at + (64 * j + lane) * VEC;
                if (k + VEC <= a.V) {
                    v[j] = *reinterpret_cast<const u32x4_a2 *>(x + k);
                    continue;
                }
                uint32_t e[VEC]; // element by element, past the end the last one's place
#pragma unroll
                for (int i = 0; i < VEC; ++i)
                    e[i] = bits_of(x[min(k + i, a.V - 1)]);
#pragma unroll
                for (int i = 0; i < VEC; ++i)
                    e[i] = k + i < a.V ? e[i] : sizeof(T) == 2 ? 0xff80u : 0xff800000u;
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    v[j][i] = sizeof(T) == 2 ? e[2 * i % VEC] | e[(2 * i + 1) % VEC] << 16 : e[i];
            }
        }
    };
    float m0 = kNegInf, m1 = kNegInf; // of every other vector of the lane's
    float m = kNegInf, sum = 0.f; // of this lane: sum of exp(x - m), 0 while there is no m
    uint32_t least = kOrderedNegInf + 1;
    int taken = 0; // of this wave
    u32x4 v[NV], next[NV];
    if (begin < end)
        load(begin, v);
    for (int at = begin, n = 1; at < end; at += STEP, ++n) {
        if (at + STEP < end)
            load(at + STEP, next);
        float half[2] = {kNegInf, kNegInf};
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int i = 0; i < VEC; i += 2)
                half[j & 1] = max3f(half[j & 1], value(v[j], i), value(v[j], i + 1));
        const float top = fmaxf(half[0], half[1]), was = m;
        m0 = fmaxf(m0, half[0]);
        m = fmaxf(m, top);
        m1 = fmaxf(m1, half[1]);
        const float ref = m == kNegInf ? 0.f : m;
        sum *= fast_exp2((was - ref) * kLog2E);
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int i = 0; i < VEC; ++i)
                sum += fast_exp2((value(v[j], i) - ref) * kLog2E);
        if ((n & (n - 1)) == 0)
            least = max(least, a.K <= 32 ? wave_kth<1>({ordered(m)}, kOrderedNegInf, 1u << 20, a.K)
                                         : wave_kth<2>({ordered(m0), ordered(m1)}, kOrderedNegInf, 1u << 20, a.K));
        const float pass = unordered(least);
        if (__builtin_amdgcn_ballot_w64(top >= pass) != 0)
#pragma unroll
            for (int j = 0; j < NV; ++j)
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    const float y = value(v[j], i);
                    const uint64_t in = __builtin_amdgcn_ballot_w64(y >= pass);
                    if (in == 0)
                        continue;
                    const int to = taken + __builtin_amdgcn_mbcnt_hi((uint32_t)(in >> 32),
                                                                     __builtin_amdgcn_mbcnt_lo((uint32_t)in, 0));
                    if (y >= pass && to < kBeamRoom)
                        room[w * kBeamRoom + to] =
                            (uint64_t)ordered(y) << 32 | ~(uint32_t)(at + (64 * j + lane) * VEC + i);
                    taken += __builtin_popcountll(in);
                }
#pragma unroll
        for (int j = 0; j < NV; ++j)
            v[j] = next[j];
    }
    const float wm = seg_all<true>(m, true), wuse = wm == kNegInf ? 0.f : wm;
    sum = seg_all<false>(sum * fast_exp2((m - wuse) * kLog2E), true); // of a lane without a logit: 0
    if (lane == 0) {
        redm[w] = wm;
        reds[w] = sum;
        redu[w] = least;
        redn[w] = taken;
    }
    __syncthreads();
    const int64_t part = (int64_t)row * a.chunks + chunk;
    if (tid == 0) {
        const float all = fmaxf(fmaxf(redm[0], redm[1]), fmaxf(redm[2], redm[3])), use = all == kNegInf ? 0.f : all;
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            s += reds[i] * fast_exp2((redm[i] - use) * kLog2E);
        a.ms[2 * part] = all;
        a.ms[2 * part + 1] = s;
    }
    least = max(max(redu[0], redu[1]), max(redu[2], redu[3]));
    for (int i = lane; i < min(taken, kBeamRoom); i += 64) {
        const uint64_t key = room[w * kBeamRoom + i];
        if (key >> 32 >= least) {
            const int to = atomicAdd(&kept, 1);
            if (to < kBeamBest)
                best[to] = key;
        }
    }
    __syncthreads();
    const int most = max(max(redn[0], redn[1]), max(redn[2], redn[3]));
    if (most > kBeamRoom || kept > kBeamBest) {
        const int last_at = min(first + 4 * a.steps * STEP, a.V);
        auto each = [&](auto &&f) {
            for (int i = first + tid; i < last_at; i += 256) {
                float y;
                if constexpr (sizeof(T) == 2)
                    y = __builtin_bit_cast(float, (uint32_t)x[i] << 16);
                else
                    y = x[i];
                f(ordered(y), (uint32_t)i);
            }
        };
        auto count = [&](auto &&f) {
            int c = 0;
            each([&](uint32_t u, uint32_t i) { c += f(u, i) ? 1 : 0; });
            return wg_sum(c, redi, tid);
        };
        // The K-th largest value, then the index up to which elements of that value belong to the K.
        uint32_t k = 0, last = 0;
        for (uint32_t bit = 0x80000000u; bit; bit >>= 1)
            if (count([&](uint32_t u, uint32_t) { return u >= (k | bit); }) >= a.K)
                k |= bit;
        const int need = a.K - count([&](uint32_t u, uint32_t) { return u > k; });
        for (uint32_t bit = 0x80000000u; bit; bit >>= 1) // the largest index before which fewer than `need` lie
            if (count([&](uint32_t u, uint32_t i) { return u == k && i < (last | bit); }) < need)
                last |= bit;
        if (tid == 0)
            kept = 0;
        __syncthreads();
        each([&](uint32_t u, uint32_t i) {
            if (u > k || (u == k && i <= last)) // K of them
                best[atomicAdd(&kept, 1) & (kBeamBest - 1)] = (uint64_t)u << 32 | ~i;
        });
        __syncthreads();
    }
    const int n = min(kept, kBeamBest);
    uint64_t *keys = a.keys + part * a.K;
    for (int i = tid; i < n; i += 256) {
        const uint64_t mine = best[i];
        int rank = 0;
#pragma unroll 8
        for (int j = 0; j < n; ++j)
            rank += best[j] > mine ? 1 : 0;
        if (rank < a.K)
            keys[rank] = mine;
    }
    for (int i = n + tid; i < a.K; i += 256)
        keys[i] = 0;
}

// ------------------------------------------------------------------------------------------
// A batch entry's K best from its beams' chunks, by ((x - m) - log sum exp(x - m)) + score in fp64, m the beam's largest
// logit (m plus the logarithm would be m alone where m is large), of equals those of the lowest beam, then the largest logit,
// then the lowest index. The chunks' lists of K are cut into segments; a thread holds the first logits of up to
// eight, and its largest gives, with the others', a threshold that at least K candidates reach. Segments whose first passes it
// are followed, and what passes counts how many are ahead. Bound by latency: one round of loads, two sums over a beam's chunks,
// a search and a count, 6 us for 1 to 64 entries of 4 to 8 beams; 13 beams over 238968 tokens, 5070 candidates, 10, and 24 where
// every candidate was looked at; 4 entries of 64 beams with K = 64 over 32000, 16384 candidates each, 3580 -> 158 with its chunks.
// ------------------------------------------------------------------------------------------
constexpr int kBeamFinalRoom = 1024;
constexpr double kLn2D = 0.693147180559945309417;

// log x of a normal x > 0: x = 2^e f with f in [sqrt(1/2), sqrt(2)], log f = 2 artanh s with s = (f - 1) / (f + 1), whose
// series s + s^3 / 3 + ... is cut where s^2 <= 0.0295 leaves less than 2^-55. In line: the library's is a call.
__device__ __forceinline__ double log_of(double x) {
    double f = __builtin_amdgcn_frexp_mant(x); // in [1/2, 1)
    int e = __builtin_amdgcn_frexp_exp(x);
    if (f < 0.707106781186547524401) {
        f *= 2.0;
        --e;
    }
    const double s = (f - 1.0) / (f + 1.0), t = s * s;
    double r = 1.0 / 19;
#pragma unroll
    for (int i = 17; i >= 1; i -= 2)
        r = fma(r, t, 1.0 / i);
    return fma((double)e, kLn2D, 2.0 * s * r);
}

__global__ __launch_bounds__(256) void attn_beam_select_kernel(const attn_beam_args a) {
    __shared__ float largest[ATTN_BEAMS_MAX];
    __shared__ double logs[ATTN_BEAMS_MAX], base[ATTN_BEAMS_MAX]; // of a done beam: 0; of one without a continuation: infinite
    __shared__ uint8_t over[ATTN_BEAMS_MAX];
    __shared__ uint64_t rv[kBeamFinalRoom], ri[kBeamFinalRoom];
    __shared__ uint32_t tops[256];
    __shared__ int from[kBeamFinalRoom], redi[4], taken; // from: the segments whose first logits are kept
    const int b = wg_id_x(), tid = wi_id_x(), lane = tid & 63;
    const int row0 = b * a.beams;
    if (tid == 0)
        taken = 0;
    // The segments' first logits are asked for at once; those of a beam without a continuation are anything. Of segment
    // s, list s mod `lists` and the s / lists-th of its segments.
    constexpr int HOLD = ATTN_BEAM_HELD / 256;
    const int lists = a.beams * a.chunks, segments = a.segments;
    const uint64_t *keys = a.keys + (int64_t)row0 * a.chunks * a.K;
    auto place = [&](int s) { // of a segment's first logit among the entry's
        const int sub = attn_div_by(s, a.by_lists);
        return (s - sub * lists) * a.K + sub * a.seg;
    };
    uint64_t held[HOLD];
#pragma unroll
    for (int r = 0; r < HOLD; ++r)
        held[r] = keys[place(min(tid + 256 * r, segments - 1))];
    // Eight lanes to a beam, whose chunks they take in turn.
    for (int i = tid >> 3; i < a.beams; i += 32) {
        const int row = row0 + i;
        const float s = a.scores[row];
        const bool done = a.done && a.done[row];
        const float *ms = a.ms + (int64_t)row * a.chunks * 2;
        auto join = [](float &m, double &sum, float m1, double s1) {
            const float both = fmaxf(m, m1), use = both == kNegInf ? 0.f : both;
            sum = sum * (double)fast_exp2((m - use) * kLog2E) + s1 * (double)fast_exp2((m1 - use) * kLog2E);
            m = both;
        };
        float m = kNegInf;
        double sum = 0.0;
#pragma unroll 4
        for (int c = tid & 7; c < a.chunks; c += 8)
            join(m, sum, ms[2 * c], ms[2 * c + 1]); // of a beam that is over: anything
#pragma unroll
        for (int j = 1; j < 8; j <<= 1) {
            const float m1 = __shfl_xor(m, j);
            const double s1 = __shfl_xor(sum, j);
            join(m, sum, m1, s1);
        }
        double l = __builtin_inf();
        if (done && finite(s))
            l = 0.0;
        else if (finite(s) && finite(m) && finite((float)sum)) // a NaN, an infinity or no logit at all: nothing
            l = log_of(sum);
        if ((tid & 7) == 0) {
            largest[i] = m;
            logs[i] = l;
            base[i] = (double)s;
            over[i] = done;
        }
    }
    __syncthreads();
    // Candidate i's score as an ordered number (0: none), and a number that is larger the further ahead it is among equal
    // ones: of the lowest beam, then the largest logit, then the lowest token.
    constexpr uint64_t LOW = ATTN_BEAM_V_MAX - 1;
    static_assert((LOW & (LOW + 1)) == 0 && LOW < 1u << 20 && ATTN_BEAMS_MAX <= 1 << 8, "60 bits");
    auto beam_of = [&](int i) { return attn_div_by(attn_div_by(i, a.by_K), a.by_chunks); };
    auto score_of = [&](int i, uint64_t key) -> uint64_t {
        const int beam = beam_of(i);
        const double l = logs[beam];
        if (ordered(l) >= ordered(__builtin_inf()))
            return 0;
        if (over[beam])
            return i == beam * a.chunks * a.K ? ordered(base[beam]) : 0;
        return key == 0 ? 0 : ordered((((double)unordered((uint32_t)(key >> 32)) - largest[beam]) - l) + base[beam]);
    };
    auto tie_of = [&](int i, uint64_t key) -> uint64_t {
        const int beam = beam_of(i);
        const uint64_t own = over[beam] ? LOW - a.done_token : key >> 32 << 20 | (LOW - ~(uint32_t)key);
        return (uint64_t)(ATTN_BEAMS_MAX - 1 - beam) << 52 | own;
    };
    // A threshold of its upper halves, which K threads' largest reach.
    uint64_t u[HOLD], top = 0;
#pragma unroll
    for (int r = 0; r < HOLD; ++r) {
        u[r] = 0;
        if (256 * r < segments) { // for all threads, or for none
            u[r] = tid + 256 * r < segments ? score_of(place(tid + 256 * r), held[r]) : 0;
            top = max(top, u[r]);
        }
    }
    tops[tid] = (uint32_t)(top >> 32);
    __syncthreads();
    const uint32_t kth = wave_kth<4>({tops[lane], tops[lane + 64], tops[lane + 128], tops[lane + 192]}, 0, 1u << 16, a.K);
    const uint64_t least = max((uint64_t)kth << 32, (uint64_t)1);
    auto keep = [&](uint64_t v, uint64_t tie) {
        const int at = atomicAdd(&taken, 1);
        if (at < kBeamFinalRoom) {
            rv[at] = v;
            ri[at] = tie;
        }
        return at;
    };
#pragma unroll
    for (int r = 0; r < HOLD; ++r)
        if (u[r] >= least) {
            const int s = tid + 256 * r, at = keep(u[r], tie_of(place(s), held[r]));
            if (at < kBeamFinalRoom)
                from[at] = s;
        }
    if (a.seg > 1) {
        // Segments whose first logit passes are followed until one does not, four logits at a time.
        __syncthreads();
        const int heads = min(taken, kBeamFinalRoom);
        __syncthreads();
        for (int h = tid; h < heads; h += 256) {
            const int s = from[h], first = place(s);
            const int end = first + min(a.seg, a.K - attn_div_by(s, a.by_lists) * a.seg);
            bool on = true;
            for (int i = first + 1; i < end && on; i += 4) {
                uint64_t next[4];
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    next[q] = keys[min(i + q, end - 1)];
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const uint64_t v = i + q < end && on ? score_of(i + q, next[q]) : 0;
                    on = v >= least;
                    if (on)
                        keep(v, tie_of(i + q, next[q]));
                }
            }
        }
    }
    __syncthreads();
    int n = taken;
    __syncthreads();
    if (n > kBeamFinalRoom) {
        // More than there is room for, by far most equal to the K-th: it is searched for bit by bit over all.
        auto each = [&](auto &&f) __attribute__((always_inline)) {
            for (int i = tid; i < lists * a.K; i += 256) {
                const uint64_t key = keys[i], v = score_of(i, key);
                if (v >= least)
                    f(v, tie_of(i, key));
            }
        };
        auto count = [&](auto &&f) {
            int c = 0;
            each([&](uint64_t v, uint64_t tie) { c += f(v, tie) ? 1 : 0; });
            return wg_sum(c, redi, tid);
        };
        uint64_t v = 0, last = 0;
        for (uint64_t bit = 1ull << 63; bit; bit >>= 1)
            if (count([&](uint64_t u, uint64_t) { return u >= (v | bit); }) >= a.K)
                v |= bit;
        const int need = a.K - count([&](uint64_t u, uint64_t) { return u > v; });
        for (uint64_t bit = 1ull << 59; bit; bit >>= 1)
            if (count([&](uint64_t u, uint64_t i) { return u == v && i >= (last | bit); }) >= need)
                last |= bit;
        if (tid == 0)
            taken = 0;
        __syncthreads();
        each([&](uint64_t x, uint64_t tie) {
            if (x > v || (x == v && tie >= last))
                keep(x, tie);
        });
        __syncthreads();
        n = min(taken, kBeamFinalRoom);
    }
    auto put = [&](int r, float score, int token, int parent) {
        const int64_t at = (int64_t)b * a.K + r;
        a.score[at] = score;
        a.token[at] = token;
        a.parent[at] = parent;
    };
    for (int i = tid; i < n; i += 256) {
        const uint64_t u = rv[i];
        const uint64_t p = ri[i];
        int rank = 0;
#pragma unroll 8
        for (int j = 0; j < n; ++j)
            rank += rv[j] > u || (rv[j] == u && ri[j] > p) ? 1 : 0;
        if (rank < a.K)
            put(rank, (float)unordered(u), (int)(LOW - (p & LOW)), row0 + ATTN_BEAMS_MAX - 1 - (int)(p >> 52));
    }
    for (int i = n + tid; i < a.K; i += 256)
        put(i, kNegInf, -1, row0);
}

// ------------------------------------------------------------------------------------------
// The paged cache's sequences follow their parents, in place. A thread holds 16 bytes at one place of the last page of
// every member of a group, or one column of their table rows: it reads them all from the parents' before it writes any, so
// that no member overwrites what another still needs. Workgroups of a group: K's, V's, their scales', the table's.
// Bound by latency for one group, and by HBM for many: what stays in place is neither read nor written. 3.2 us for four
// beams of 777 tokens, 9.6 for 48 groups of five of 1000 in 4 bits, 8 heads of 128.
// ------------------------------------------------------------------------------------------
template <int NB> __global__ __launch_bounds__(256) void attn_kv_reorder_kernel(const attn_reorder_args a) {
    const int per = attn_reorder_wgs(&a), g = uniform(wg_id_x() / per), tid = wi_id_x();
    int wg = wg_id_x() - g * per;
    const int first = (a.first + g) * a.beams;
    const int64_t most = (int64_t)a.cols << a.lgp;
    const int len = (int)min((int64_t)max(scalar_i32(a.kv_len, first), 0), most);
    const int full = len >> a.lgp, rest = len & ((1 << a.lgp) - 1);
    int par[NB];
#pragma unroll
    for (int i = 0; i < NB; ++i)
        par[i] = i < a.beams ? attn_parent_of(scalar_i32(a.parent, first + i), first, i, a.beams) : i;
    int32_t *table = a.table + (int64_t)first * a.cols;
    if (wg >= 2 * (a.data_wgs + a.scale_wgs)) {
        wg -= 2 * (a.data_wgs + a.scale_wgs);
        for (int c = wg * 256 + tid; c < full; c += a.table_wgs * 256) {
            int32_t x[NB];
#pragma unroll
            for (int i = 0; i < NB; ++i)
                if (par[i] != i)
                    x[i] = table[(int64_t)par[i] * a.cols + c];
#pragma unroll
            for (int i = 0; i < NB; ++i)
                if (par[i] != i)
                    table[(int64_t)i * a.cols + c] = x[i];
        }
        return;
    }
    if (rest == 0)
        return;
    const bool scales = wg >= 2 * a.data_wgs;
    if (scales)
        wg -= 2 * a.data_wgs;
    const int wgs = scales ? a.scale_wgs : a.data_wgs, row = scales ? a.srow : a.row;
    const bool v = wg >= wgs;
    uint8_t *pool = scales ? (v ? a.vs : a.ks) : (v ? a.v : a.k);
    const int units = (row << a.lgp) / 16; // of a head's rows in a page
    const int at = (wg - (v ? wgs : 0)) * 256 + tid, h = at / units, off = (at - h * units) * 16;
    if (h >= a.Hkv || off >= rest * row)
        return;
    const int64_t page = (int64_t)a.Hkv * row << a.lgp, in = ((int64_t)h * row << a.lgp) + off;
    // The column of the last page is none that this call writes.
    int pg[NB];
    u32x4 x[NB];
#pragma unroll
    for (int i = 0; i < NB; ++i) {
        pg[i] = -1;
        if (par[i] == i)
            continue;
        const int src = scalar_i32(table, (int64_t)par[i] * a.cols + full);
        pg[i] = attn_page_ok(src, a.pages) ? scalar_i32(table, (int64_t)i * a.cols + full) : -1;
        if (attn_page_ok(pg[i], a.pages))
            x[i] = *reinterpret_cast<const u32x4 *>(pool + src * page + in);
    }
#pragma unroll
    for (int i = 0; i < NB; ++i)
        if (attn_page_ok(pg[i], a.pages))
            *reinterpret_cast<u32x4 *>(pool + pg[i] * page + in) = x[i];
}

} // namespace

extern "C" int attn_hip_launch_beam(const struct attn_beam_args *ap, int bits, void *stream) {
    const attn_beam_args &a = *ap;
    const hipStream_t st = (hipStream_t)stream;
    const int64_t grid = (int64_t)a.B * a.beams * a.chunks;
    if (grid <= 0 || grid > 0x7fffffff || a.beams > ATTN_BEAMS_MAX || a.K > ATTN_BEAM_K_MAX ||
        (int64_t)a.chunks * a.steps * 4 * ATTN_BEAM_STEP(bits / 8) < a.V || a.segments > ATTN_BEAM_HELD)
        return (int)hipErrorInvalidValue;
    const dim3 g((unsigned)grid), block(256);
    if (bits == 16)
        hipLaunchKernelGGL(attn_beam_chunk_kernel<uint16_t>, g, block, 0, st, a);
    else
        hipLaunchKernelGGL(attn_beam_chunk_kernel<float>, g, block, 0, st, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess)
        return (int)e;
    hipLaunchKernelGGL(attn_beam_select_kernel, dim3((unsigned)a.B), block, 0, st, a);
    return (int)hipGetLastError();
}

extern "C" int attn_hip_launch_reorder(const struct attn_reorder_args *ap, void *stream) {
    const attn_reorder_args &a = *ap;
    const int64_t grid = (int64_t)a.groups * attn_reorder_wgs(&a);
    if (grid <= 0 || grid > ATTN_REORDER_GRID || a.beams < 1 || a.beams > ATTN_REORDER_MAX)
        return (int)hipErrorInvalidValue;
    const dim3 g((unsigned)grid), block(256);
    const hipStream_t st = (hipStream_t)stream;
    if (a.beams <= 4)
        hipLaunchKernelGGL(attn_kv_reorder_kernel<4>, g, block, 0, st, a);
    else if (a.beams <= 8)
        hipLaunchKernelGGL(attn_kv_reorder_kernel<8>, g, block, 0, st, a);
    else if (a.beams <= 16)
        hipLaunchKernelGGL(attn_kv_reorder_kernel<16>, g, block, 0, st, a);
    else
        hipLaunchKernelGGL(attn_kv_reorder_kernel<32>, g, block, 0, st, a);
    return (int)hipGetLastError();
}

#endif
