// attn_beam_kernels.h -- gfx950 kernels of beam search: the K best continuations of each batch entry's beams over the
// vocabulary (attn_beam_select), and the paged cache's sequences following their parents (attn_kv_reorder). Part of
// attn_kernels.hip.
#ifndef ATTN_BEAM_KERNELS_H
#define ATTN_BEAM_KERNELS_H

#include "attn_beam_rule.h"
#include "attn_device.h"
#include "attn_launch.h"

namespace {

// Floats and doubles as unsigned numbers of the same order; 0 stands for none (a NaN with the sign bit).
__device__ __forceinline__ uint32_t ordered(float x) {
    const uint32_t u = __builtin_bit_cast(uint32_t, x);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float unordered(uint32_t u) {
    return __builtin_bit_cast(float, u & 0x80000000u ? u & 0x7fffffffu : ~u);
}
__device__ __forceinline__ uint64_t ordered(double x) {
    const uint64_t u = __builtin_bit_cast(uint64_t, x);
    return u >> 63 ? ~u : u | 0x8000000000000000ull;
}
__device__ __forceinline__ double unordered(uint64_t u) {
    return __builtin_bit_cast(double, u >> 63 ? u & 0x7fffffffffffffffull : ~u);
}
constexpr uint32_t kOrderedNegInf = 0x007fffffu; // ordered(-inf): what is above it is a candidate
// A test of the bits, which the compiler must not see as one of a float: those are compiled as if there were no NaN.
__device__ __forceinline__ bool finite(float x) {
    return (opaque(__builtin_bit_cast(uint32_t, x)) & 0x7f800000u) != 0x7f800000u;
}

// A value that at least K of the wave's lanes reach (the lowest one where fewer are above `none`), and hardly more: the
// interval between the smallest and the largest is halved until the count is between K and K + 7.
template <typename U> __device__ __forceinline__ U wave_kth(U x, U none, int K) {
    U lo = none, hi = ~(U)0; // count(>= lo) >= K or lo == none; count(>= hi) < K or unknown
    if (__builtin_popcountll(__builtin_amdgcn_ballot_w64(x > none)) < K)
        return none;
    while (lo + 1 < hi) {
        const U mid = lo + (hi - lo) / 2;
        const int n = __builtin_popcountll(__builtin_amdgcn_ballot_w64(x >= mid));
        if (n >= K) {
            lo = mid;
            if (n < K + 8)
                break;
        } else {
            hi = mid;
        }
    }
    return lo;
}

__device__ __forceinline__ uint32_t bits_lo(uint64_t x) { return (uint32_t)x; }

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
// One chunk of a row: its maximum m and sum of e^(x - m), and its K largest logits, of equals those at the lowest index.
// Each thread holds its elements in registers. The threads' own maxima give a threshold that at least K elements reach
// (wave_kth, the largest of four waves); what reaches it goes to LDS, a few dozen elements, and each counts how many
// are ahead of it. Where more reach it than LDS has room for (equal logits) the K-th element's value and index are
// searched for bit by bit. HBM-bound: each logit is read once.
// ------------------------------------------------------------------------------------------
constexpr int kBeamRoom = 512;

template <typename T, int EPT> __global__ __launch_bounds__(256) void attn_beam_chunk_kernel(const attn_beam_args a) {
    constexpr int VEC = 16 / sizeof(T), NVEC = EPT / VEC;
    typedef T __attribute__((ext_vector_type(VEC), aligned(sizeof(T)))) vec;
    __shared__ uint64_t room[kBeamRoom];
    __shared__ float redf[4];
    __shared__ uint32_t redu[4];
    __shared__ int redi[4], taken;
    const int row = wg_id_x() / a.chunks, chunk = wg_id_x() - row * a.chunks, tid = wi_id_x(), w = tid >> 6;
    if ((a.done && a.done[row]) || !finite(a.scores[row]))
        return;
    const T *x = reinterpret_cast<const T *>(a.logits) + row * a.row;
    const int first = chunk * 256 * EPT;
    float e[EPT];
    auto value = [](T t) {
        if constexpr (sizeof(T) == 2)
            return __builtin_bit_cast(float, (uint32_t)t << 16);
        else
            return t;
    };
    // Element i of vector j has index first + (256 j + tid) VEC + i.
#pragma unroll
    for (int j = 0; j < NVEC; ++j) {
        const int at = first + (256 * j + tid) * VEC;
        if (at + VEC <= a.V) {
            const vec v = __builtin_nontemporal_load(reinterpret_cast<const vec *>(x + at));
#pragma unroll
            for (int i = 0; i < VEC; ++i)
                e[VEC * j + i] = value(v[i]);
        } else {
#pragma unroll
            for (int i = 0; i < VEC; ++i)
                e[VEC * j + i] = at + i < a.V ? value(x[at + i]) : kNegInf;
        }
    }
    if (tid == 0)
        taken = 0;
    uint32_t top = 0; // a NaN's bits are above infinity's, or lowest of all; either makes the sum one
    float mx = kNegInf;
#pragma unroll
    for (int i = 0; i < EPT; ++i)
        mx = fmaxf(mx, e[i]);
    top = ordered(mx);
    const uint32_t kth = wave_kth<uint32_t>(top, kOrderedNegInf, a.K);
    float m = mx;
    m = seg_all<true>(m, true);
    if ((tid & 63) == 0) {
        redf[w] = m;
        redu[w] = kth;
    }
    __syncthreads();
    m = fmaxf(fmaxf(redf[0], redf[1]), fmaxf(redf[2], redf[3]));
    const uint32_t least = max(max(max(redu[0], redu[1]), max(redu[2], redu[3])), kOrderedNegInf + 1);
    if (top >= least)
#pragma unroll
        for (int i = 0; i < EPT; ++i) {
            const uint32_t u = ordered(e[i]);
            if (u >= least) {
                const int at = atomicAdd(&taken, 1);
                if (at < kBeamRoom)
                    room[at] = (uint64_t)u << 32 | ~(uint32_t)(first + (256 * (i / VEC) + tid) * VEC + i % VEC);
            }
        }
    const float muse = m == kNegInf ? 0.f : m;
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < EPT; ++i)
        sum += fast_exp2((e[i] - muse) * 1.44269504088896341f);
    sum = seg_all<false>(sum, true);
    __syncthreads();
    if ((tid & 63) == 0)
        redf[w] = sum;
    int n = taken;
    __syncthreads();
    const int64_t part = (int64_t)row * a.chunks + chunk;
    if (tid == 0) {
        a.ms[2 * part] = m;
        a.ms[2 * part + 1] = redf[0] + redf[1] + redf[2] + redf[3];
    }
    if (n > kBeamRoom) {
        // The K-th largest value, then the index up to which elements of that value belong to the K.
        auto count = [&](auto &&f) {
            int c = 0;
#pragma unroll
            for (int i = 0; i < EPT; ++i)
                c += f(ordered(e[i]), (uint32_t)(first + (256 * (i / VEC) + tid) * VEC + i % VEC)) ? 1 : 0;
            return wg_sum(c, redi, tid);
        };
        uint32_t v = 0, last = 0;
        for (uint32_t bit = 0x80000000u; bit; bit >>= 1)
            if (count([&](uint32_t u, uint32_t) { return u >= (v | bit); }) >= a.K)
                v |= bit;
        const int need = a.K - count([&](uint32_t u, uint32_t) { return u > v; });
        for (uint32_t bit = 0x80000000u; bit; bit >>= 1) // the largest index before which fewer than `need` lie
            if (count([&](uint32_t u, uint32_t i) { return u == v && i < (last | bit); }) < need)
                last |= bit;
        if (tid == 0)
            taken = 0;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < EPT; ++i) {
            const uint32_t u = ordered(e[i]), at = first + (256 * (i / VEC) + tid) * VEC + i % VEC;
            if (u > v || (u == v && at <= last)) // K of them
                room[atomicAdd(&taken, 1) & (kBeamRoom - 1)] = (uint64_t)u << 32 | ~at;
        }
        __syncthreads();
        n = min(taken, kBeamRoom);
    }
    uint64_t *keys = a.keys + part * a.K;
    for (int i = tid; i < n; i += 256) {
        const uint64_t mine = room[i];
        int rank = 0;
        for (int j = 0; j < n; ++j)
            rank += room[j] > mine ? 1 : 0;
        if (rank < a.K)
            keys[rank] = mine;
    }
    for (int i = n + tid; i < a.K; i += 256)
        keys[i] = 0;
}

// ------------------------------------------------------------------------------------------
// A batch entry's K best from its beams' chunks, by (x - lse) + score in fp64, of equals those of the lowest beam and
// index. The chunks' lists are sorted: their heads give a threshold that at least K candidates reach, each list is
// followed down to it, and what reaches it counts how many are ahead.
// ------------------------------------------------------------------------------------------
constexpr int kBeamFinalRoom = 1024;
constexpr int kBeamMax = 256;

__global__ __launch_bounds__(256) void attn_beam_select_kernel(const attn_beam_args a) {
    __shared__ double lse[kBeamMax], base[kBeamMax]; // lse of a done beam: 0, of one that offers nothing: infinite
    __shared__ uint64_t rv[kBeamFinalRoom], redu[4];
    __shared__ uint32_t ri[kBeamFinalRoom];
    __shared__ int redi[4], taken;
    const int b = wg_id_x(), tid = wi_id_x(), w = tid >> 6, lane = tid & 63;
    const int row0 = b * a.beams;
    if (tid == 0)
        taken = 0;
    for (int i = w; i < a.beams; i += 4) {
        const int row = row0 + i;
        const float s = a.scores[row];
        const bool done = a.done && a.done[row];
        double l = __builtin_inf();
        if (done && finite(s)) {
            l = 0.0;
        } else if (finite(s)) {
            const float *ms = a.ms + (int64_t)row * a.chunks * 2;
            float m = kNegInf;
            for (int c = lane; c < a.chunks; c += 64)
                m = fmaxf(m, ms[2 * c]);
            m = seg_all<true>(m, true);
            const float muse = m == kNegInf ? 0.f : m;
            double sum = 0.0;
            for (int c = lane; c < a.chunks; c += 64)
                sum += (double)ms[2 * c + 1] * (double)fast_exp2((ms[2 * c] - muse) * 1.44269504088896341f);
#pragma unroll
            for (int j = 1; j < 64; j <<= 1)
                sum += __shfl_xor(sum, j);
            // A NaN, an infinity or no logit at all: the beam offers nothing.
            if (finite(m) && finite((float)sum))
                l = (double)m + log(sum);
        }
        if (lane == 0) {
            lse[i] = l;
            base[i] = (double)s;
        }
    }
    __syncthreads();
    const int lists = a.beams * a.chunks;
    // Candidate r of list i: its score as an ordered number (0: none) and its place among the entry's candidates.
    auto candidate = [&](int i, int r, uint32_t &place) -> uint64_t {
        const int beam = i / a.chunks, row = row0 + beam;
        const double l = lse[beam];
        if (ordered(l) >= ordered(__builtin_inf()))
            return 0;
        if (a.done && a.done[row]) {
            place = (uint32_t)beam * a.V + a.done_token;
            return r == 0 && i == beam * a.chunks ? ordered(base[beam]) : 0;
        }
        const uint64_t key = a.keys[((int64_t)row0 * a.chunks + i) * a.K + r];
        if (key == 0)
            return 0;
        place = (uint32_t)beam * a.V + ~bits_lo(key);
        return ordered(((double)unordered((uint32_t)(key >> 32)) - l) + base[beam]);
    };
    uint64_t top = 0;
    uint32_t place = 0;
    for (int i = tid; i < lists; i += 256)
        top = max(top, candidate(i, 0, place));
    const uint64_t kth = wave_kth<uint64_t>(top, 0, a.K);
    if (lane == 0)
        redu[w] = kth;
    __syncthreads();
    uint64_t least = max(max(max(redu[0], redu[1]), max(redu[2], redu[3])), (uint64_t)1);
    auto collect = [&](auto &&f) {
        for (int i = tid; i < lists; i += 256)
            for (int r = 0; r < a.K; ++r) {
                const uint64_t u = candidate(i, r, place);
                if (u < least)
                    break;
                if (f(u, place)) {
                    const int at = atomicAdd(&taken, 1);
                    if (at < kBeamFinalRoom) {
                        rv[at] = u;
                        ri[at] = place;
                    }
                }
            }
        __syncthreads();
    };
    collect([](uint64_t, uint32_t) { return true; });
    int n = taken;
    __syncthreads();
    if (n > kBeamFinalRoom) {
        auto count = [&](auto &&f) {
            int c = 0;
            for (int i = tid; i < lists; i += 256)
                for (int r = 0; r < a.K; ++r) {
                    const uint64_t u = candidate(i, r, place);
                    if (u < least)
                        break;
                    c += f(u, place) ? 1 : 0;
                }
            return wg_sum(c, redi, tid);
        };
        uint64_t v = 0;
        uint32_t last = 0;
        for (uint64_t bit = 1ull << 63; bit; bit >>= 1)
            if (count([&](uint64_t u, uint32_t) { return u >= (v | bit); }) >= a.K)
                v |= bit;
        const int need = a.K - count([&](uint64_t u, uint32_t) { return u > v; });
        for (uint32_t bit = 0x80000000u; bit; bit >>= 1)
            if (count([&](uint64_t u, uint32_t i) { return u == v && i < (last | bit); }) < need)
                last |= bit;
        if (tid == 0)
            taken = 0;
        __syncthreads();
        collect([&](uint64_t u, uint32_t i) { return u > v || (u == v && i <= last); });
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
        const uint32_t p = ri[i];
        int rank = 0;
        for (int j = 0; j < n; ++j)
            rank += rv[j] > u || (rv[j] == u && ri[j] < p) ? 1 : 0;
        if (rank < a.K)
            put(rank, (float)unordered(u), (int)(p % (uint32_t)a.V), row0 + (int)(p / (uint32_t)a.V));
    }
    for (int i = n + tid; i < a.K; i += 256)
        put(i, kNegInf, -1, row0);
}

// ------------------------------------------------------------------------------------------
// The paged cache's sequences follow their parents, in place. A thread holds 16 bytes at one place of the last page of
// every member of a group, or one column of their table rows: it reads them all from the parents' before it writes any, so
// that no member overwrites what another still needs. Workgroups of a group: K's, V's, their scales', the table's.
// Bound by latency for one group, and by HBM for many: what stays in place is neither read nor written.
// ------------------------------------------------------------------------------------------
template <int NB> __global__ __launch_bounds__(256) void attn_kv_reorder_kernel(const attn_reorder_args a) {
    const int per = 2 * (a.data_wgs + a.scale_wgs) + a.table_wgs;
    const int g = uniform(wg_id_x() / per), tid = wi_id_x();
    int wg = wg_id_x() - g * per;
    const int first = g * a.beams;
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

extern "C" int attn_hip_launch_beam(const struct attn_beam_args *ap, int bits, int chunk, void *stream) {
    const attn_beam_args &a = *ap;
    const hipStream_t st = (hipStream_t)stream;
    const int64_t grid = (int64_t)a.B * a.beams * a.chunks;
    if (grid <= 0 || grid > 0x7fffffff || a.beams > kBeamMax || a.K > 64 || (int64_t)a.chunks * chunk < a.V)
        return (int)hipErrorInvalidValue;
    const dim3 g((unsigned)grid), block(256);
    if (chunk == ATTN_BEAM_CHUNK) {
        if (bits == 16)
            hipLaunchKernelGGL((attn_beam_chunk_kernel<uint16_t, ATTN_BEAM_CHUNK / 256>), g, block, 0, st, a);
        else
            hipLaunchKernelGGL((attn_beam_chunk_kernel<float, ATTN_BEAM_CHUNK / 256>), g, block, 0, st, a);
    } else {
        if (bits == 16)
            hipLaunchKernelGGL((attn_beam_chunk_kernel<uint16_t, ATTN_BEAM_CHUNK_SMALL / 256>), g, block, 0, st, a);
        else
            hipLaunchKernelGGL((attn_beam_chunk_kernel<float, ATTN_BEAM_CHUNK_SMALL / 256>), g, block, 0, st, a);
    }
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess)
        return (int)e;
    hipLaunchKernelGGL(attn_beam_select_kernel, dim3((unsigned)a.B), block, 0, st, a);
    return (int)hipGetLastError();
}

extern "C" int attn_hip_launch_reorder(const struct attn_reorder_args *ap, void *stream) {
    const attn_reorder_args &a = *ap;
    const int64_t grid = (int64_t)a.groups * (2 * (a.data_wgs + a.scale_wgs) + a.table_wgs);
    if (grid <= 0 || grid > 0x7fffffff || a.beams < 1 || a.beams > 32)
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
