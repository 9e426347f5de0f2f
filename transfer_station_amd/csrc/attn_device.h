// attn_device.h -- device helpers shared by this library's gfx950 kernels: ids, vector types, loads at
// any alignment, lane exchanges, buffer descriptors and LDS-DMA. Included by attn_kernels.hip.
#ifndef ATTN_DEVICE_H
#define ATTN_DEVICE_H

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>
#include <utility>

namespace {

typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;
typedef __attribute__((ext_vector_type(4))) short s16x4;
typedef __attribute__((ext_vector_type(16))) float f32x16;
typedef __attribute__((ext_vector_type(4))) float f32x4;
typedef __attribute__((ext_vector_type(4))) uint32_t u32x4;
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

constexpr float kNegInf = -__builtin_inff();

// Workgroup and work-item ids read straight from their registers. HIP's blockIdx / threadIdx /
// gridDim go through device-library functions that are built with IEEE mode on; this library
// is built with it off (-mno-amdgpu-ieee), so the compiler will not inline them, and each use
// would be an out-of-line call in the kernel's prologue. The workgroup count comes from the
// kernel's own arguments instead: reading the grid size from the dispatch packet
// (__builtin_amdgcn_grid_size_x) in every workgroup's prologue measured 2-22% slower.
// The two kernels that stage tiles by LDS-DMA (the fast prefill and the V^T decode) still take
// threadIdx.x, and with it one such call, on purpose. In a kernel without any call this
// compiler makes each LDS read of a tile wait (vmcnt) for the DMA of the next tile into the
// other buffer, which it cannot tell apart from this one: measured 3-15% slower on the prefill
// shapes. With the call it leaves that ordering to the kernel, which does it itself (each wave
// waits for its own DMA, vmcnt(0), before the barrier that ends a tile).
__device__ __forceinline__ int wg_id_x() { return (int)__builtin_amdgcn_workgroup_id_x(); }
__device__ __forceinline__ int wg_id_y() { return (int)__builtin_amdgcn_workgroup_id_y(); }
__device__ __forceinline__ int wg_id_z() { return (int)__builtin_amdgcn_workgroup_id_z(); }
__device__ __forceinline__ int wi_id_x() { return (int)__builtin_amdgcn_workitem_id_x(); }

// Workgroups are dispatched round-robin over the 8 XCDs (each with its own L2). Remap the
// hardware block id so that consecutive logical ids land on the same XCD: logical ids that
// share a kv head then share that XCD's L2 copy of K/V.
__device__ __forceinline__ int xcd_remap(int b, int n) {
    const int per = n >> 3, rem = n & 7;
    const int x = b & 7, i = b >> 3;
    return (x < rem) ? x * (per + 1) + i : rem * (per + 1) + (x - rem) * per + i;
}

// xcd_remap for a grid resident all at once at two workgroups per CU (n <= 2 * CUs). Each
// XCD hands its blocks to its R CUs in order, one slot per CU first, so XCD positions i and
// i + R share a CU (measured with a HW_ID probe: blocks b and b + 256 on MI355X). Reversing
// positions [R, n_x) pairs the first round's heaviest item with the second round's lightest,
// when the logical order is heaviest first. R = 0 gives xcd_remap.
__device__ __forceinline__ int xcd_remap_paired(int b, int n, int R) {
    const int per = n >> 3, rem = n & 7;
    const int x = b & 7, nx = (x < rem) ? per + 1 : per;
    int i = b >> 3;
    if (R > 0 && i >= R)
        i = R + (nx - 1 - i);
    return (x < rem) ? x * (per + 1) + i : rem * (per + 1) + (x - rem) * per + i;
}

// f(std::integral_constant<int, 0>{}), ..., f(std::integral_constant<int, N-1>{}): an unrolled loop
// whose index is a constant expression (needed for sched_group_barrier counts).
template <typename F, int... I>
__device__ __forceinline__ void static_for_impl(F &&f, std::integer_sequence<int, I...>) {
    (f(std::integral_constant<int, I>{}), ...);
}
template <int N, typename F> __device__ __forceinline__ void static_for(F &&f) {
    static_for_impl(f, std::make_integer_sequence<int, N>{});
}

__device__ __forceinline__ u32x4 zero4() {
    u32x4 z = {0u, 0u, 0u, 0u};
    return z;
}

// Unaligned vectors: gfx950 serves 16-byte global accesses at any element alignment, so tensors
// whose rows are not 16-byte aligned are read 16 bytes at a time too (element-wise loads, eight
// 2-byte loads and their packing per chunk, made such calls 6-15x slower). O is fp32: 4-aligned.
typedef u32x4 __attribute__((aligned(2))) u32x4_a2;
typedef f32x4 __attribute__((aligned(4))) f32x4_a4;

template <bool NT> __device__ __forceinline__ u32x4 load16_any(const uint16_t *p) {
    return NT ? __builtin_nontemporal_load(reinterpret_cast<const u32x4_a2 *>(p))
              : *reinterpret_cast<const u32x4_a2 *>(p);
}

// x as a value that the compiler takes for new here: what follows from it is computed where it is
// used, not hoisted out of the key loop and spilled.
__device__ __forceinline__ uint32_t opaque(uint32_t x) {
    asm volatile("" : "+v"(x));
    return x;
}

// v without its first n (0..8) of eight 16-bit elements, zeros behind.
__device__ __forceinline__ u32x4 drop_elems(u32x4 v, int n) {
    const int h = (n & 1) * 16;
    const bool n2 = n & 2, n4 = n & 4, n8 = n & 8;
    const uint32_t a0 = __builtin_amdgcn_alignbit(v[1], v[0], h);
    const uint32_t a1 = __builtin_amdgcn_alignbit(v[2], v[1], h);
    const uint32_t a2 = __builtin_amdgcn_alignbit(v[3], v[2], h), a3 = v[3] >> h;
    const uint32_t b0 = n2 ? a1 : a0, b1 = n2 ? a2 : a1, b2 = n2 ? a3 : a2, b3 = n2 ? 0u : a3;
    return u32x4{n8 ? 0u : n4 ? b2 : b0, n8 ? 0u : n4 ? b3 : b1, n4 || n8 ? 0u : b2,
                 n4 || n8 ? 0u : b3};
}

// Elements [i, i+8) of the n-element row at p one by one, zero-filled past n: rows of fewer than
// eight elements. load_rolled does it in a loop: code that hardly any call reaches.
__device__ __forceinline__ u32x4 load_short(const uint16_t *p, int i, int n) {
    if (i >= n)
        return zero4();
    uint32_t e[8];
#pragma unroll
    for (int j = 0; j < 8; ++j)
        e[j] = i + j < n ? (uint32_t)p[i + j] : 0u;
    return u32x4{e[0] | (e[1] << 16), e[2] | (e[3] << 16), e[4] | (e[5] << 16), e[6] | (e[7] << 16)};
}

__device__ __forceinline__ u32x4 load_rolled(const uint16_t *p, int i, int n) {
    u32x4 v = zero4();
#pragma unroll 1
    for (int j = min(n, i + 8) - 1; j >= i; --j)
        v = u32x4{(v[0] << 16) | p[j], __builtin_amdgcn_alignbit(v[1], v[0], 16),
                  __builtin_amdgcn_alignbit(v[2], v[1], 16),
                  __builtin_amdgcn_alignbit(v[3], v[2], 16)};
    return v;
}

// The first m (1..7) of eight 16-bit elements, zeros behind.
__device__ __forceinline__ u32x4 keep_elems(u32x4 v, int m) {
    auto w = [&](uint32_t x, int j) {
        return m >= 2 * j + 2 ? x : m == 2 * j + 1 ? x & 0xffffu : 0u;
    };
    return u32x4{w(v[0], 0), w(v[1], 1), w(v[2], 2), w(v[3], 3)};
}

// Elements [i, i+8) of the n-element row at p (n >= 8), at any alignment and without a read outside
// the row, in two steps: load_piece reads a piece that reaches past the row's end as its last
// eight elements, and trim_piece shifts it where it is used, zeros behind (a shift at the load
// would wait for it before the next piece's load is issued). Pieces past the end are zeros. ie
// (wave-uniform) bounds the elements of the wave's lanes.
template <bool NT = false>
__device__ __forceinline__ u32x4 load_piece(const uint16_t *p, int i, int n, int ie) {
    if (i >= n)
        return zero4();
    if ((n & 7) != 0 && ie > n)
        return load16_any<NT>(p + min(i, n - 8));
    return load16_any<NT>(p + i);
}

__device__ __forceinline__ u32x4 trim_piece(u32x4 v, int i, int n, int ie) {
    return (n & 7) != 0 && ie > n ? drop_elems(v, (int)opaque(min(max(i + 8 - n, 0), 8))) : v;
}

// Aligned tensors: eight consecutive bf16 of one row, columns [col, col+8), zero-filled past D or
// when !ok. D % 8 == 0 and a 16-byte aligned base, so one 16-byte load covers them.
// NT marks the load non-temporal (data read once: HBM streams such loads ≈ 15% faster).
template <bool NT = false>
__device__ __forceinline__ u32x4 load_row8(const uint16_t *base, size_t row, int col, int D,
                                           bool ok) {
    if (!ok || col >= D)
        return zero4();
    const uint16_t *p = base + row * (size_t)D + col;
    return NT ? __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(p))
              : *reinterpret_cast<const u32x4 *>(p);
}

// Aligned tensors: eight consecutive keys [key, key+8) of row d of a V^T head ([D][Sk], row stride
// Sk), zero-filled at d >= D or key >= klim. Sk % 8 == 0 and a 16-byte aligned base (with
// key % 8 == 0 and klim % 8 == 0 a chunk is then wholly inside or wholly outside).
template <bool NT = false>
__device__ __forceinline__ u32x4 load_vt8(const uint16_t *base, int d, int key, int Sk, int D,
                                          int klim) {
    if (d >= D || key >= klim)
        return zero4();
    const uint16_t *p = base + (size_t)d * Sk + key;
    return NT ? __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(p))
              : *reinterpret_cast<const u32x4 *>(p);
}

__device__ __forceinline__ bf16x8 as_bf16x8(u32x4 v) { return __builtin_bit_cast(bf16x8, v); }

__device__ __forceinline__ bf16x8 join_tr(s16x4 lo, s16x4 hi) {
    typedef __attribute__((ext_vector_type(8))) short s16x8;
    s16x8 r = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
    return __builtin_bit_cast(bf16x8, r);
}

// ds_read_b64_tr_b16: within each 16-lane group, lane i receives element r (r = 0..3) from
// row (4r + i/4) of the group's 16x4 matrix of 8-byte reads, element i%4. Lanes that address
// V[key0 + j/4][d0 + 4*(j%4)] therefore receive V[key0 + r][d0 + i]: four keys for one column.
__device__ __forceinline__ s16x4 lds_read_tr(const uint16_t *p) {
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)(p));
}

__device__ __forceinline__ float fast_exp2(float x) { return __builtin_amdgcn_exp2f(x); }

// max(a, b, c); with IEEE mode off the compiler emits v_max3_f32 or two v_max_f32. No inline
// asm here on purpose: these read MFMA results, and a VALU read of an MFMA result needs wait
// states that the hardware does not enforce; the compiler inserts them only for instructions it
// can see (an asm v_max3 right after the last Q.K^T MFMA read stale scores).
__device__ __forceinline__ float max3f(float a, float b, float c) { return fmaxf(fmaxf(a, b), c); }

// max(x[lane], x[lane ^ 32]), through ds_bpermute (compiler-managed waits). The row max runs on
// an item's first key tile and on rare recomputed tiles only, so the exchange's cost is small.
// Lane exchanges of a value with lane l ^ 16 or l ^ 32 on the VALU (v_permlane16_swap /
// v_permlane32_swap with the value as both operands), where __shfl_xor goes through the LDS
// crossbar and its wait (lgkmcnt) also waits for the wave's LDS reads in flight. Each lane gets
// the pair {its value, its partner's} in one order or the other, so max and sum (commutative)
// give exactly what fmaxf / + with the shuffled value give.
__device__ __forceinline__ float max_xor32(float x) {
    const unsigned u = __builtin_bit_cast(unsigned, x);
    const auto p = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    return fmaxf(__builtin_bit_cast(float, (unsigned)p[0]), __builtin_bit_cast(float, (unsigned)p[1]));
}
__device__ __forceinline__ float sum_xor32(float x) {
    const unsigned u = __builtin_bit_cast(unsigned, x);
    const auto p = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    return __builtin_bit_cast(float, (unsigned)p[0]) + __builtin_bit_cast(float, (unsigned)p[1]);
}
__device__ __forceinline__ float max_xor16(float x) {
    const unsigned u = __builtin_bit_cast(unsigned, x);
    const auto p = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    return fmaxf(__builtin_bit_cast(float, (unsigned)p[0]), __builtin_bit_cast(float, (unsigned)p[1]));
}
__device__ __forceinline__ float sum_xor16(float x) {
    const unsigned u = __builtin_bit_cast(unsigned, x);
    const auto p = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    return __builtin_bit_cast(float, (unsigned)p[0]) + __builtin_bit_cast(float, (unsigned)p[1]);
}

__device__ __forceinline__ void lds_wave_fence() {
    // Wave-private LDS reuse: finish this wave's outstanding LDS traffic and keep the compiler
    // from moving LDS accesses across this point.
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
}

// The descriptor must live in scalar registers; its inputs are workgroup-uniform, and the
// readfirstlane makes that explicit so the compiler never falls back to a per-lane loop.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t make_rsrc(const void *base, uint32_t bytes) {
    const uint64_t a = reinterpret_cast<uint64_t>(base);
    const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)a);
    const uint32_t hi = __builtin_amdgcn_readfirstlane((uint32_t)(a >> 32));
    void *p = reinterpret_cast<void *>(((uint64_t)hi << 32) | lo);
    return __builtin_amdgcn_make_buffer_rsrc(p, (short)0, (int)__builtin_amdgcn_readfirstlane(bytes),
                                             0x00020000);
}

// LDS-DMA: 16 bytes per lane from buffer r at byte voff + IMM straight into LDS, lane i writing
// [lds + IMM + 16 i, +16) (the immediate offset moves both addresses; lds must be wave-uniform).
// Bytes past the buffer's range arrive as zero. Completion is counted by vmcnt.
// AUX is the cache policy: 0 ordinary, kDmaNT non-temporal (data read once).
constexpr int kDmaNT = 2;
template <int IMM, int AUX = 0>
__device__ __forceinline__ void dma16(__amdgpu_buffer_rsrc_t r, uint16_t *lds, uint32_t voff) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void *)lds, 16,
                                             voff, 0, IMM, AUX);
}

// s_waitcnt operand (gfx9 encoding) that waits until at most n vector memory operations of
// the wave are in flight, with no wait on expcnt or lgkmcnt.
constexpr int waitcnt_vm(int n) { return 0x0F70 | (n & 15) | ((n >> 4) << 14); }

// max or sum over each 16 (all: 64) lanes of the wave, in every lane, on the VALU.
template <bool MAX> __device__ __forceinline__ float seg_all(float x, bool all) {
    auto op = [](float a, float b) { return MAX ? fmaxf(a, b) : a + b; };
    auto ror = [](float v, auto C) {
        const int u = __builtin_bit_cast(int, v);
        return __builtin_bit_cast(
            float, __builtin_amdgcn_update_dpp(u, u, decltype(C)::value, 0xf, 0xf, false));
    };
    x = op(x, ror(x, std::integral_constant<int, 0x128>{})); // row_ror:8, 4, 2, 1
    x = op(x, ror(x, std::integral_constant<int, 0x124>{}));
    x = op(x, ror(x, std::integral_constant<int, 0x122>{}));
    x = op(x, ror(x, std::integral_constant<int, 0x121>{}));
    if (all)
        x = MAX ? max_xor32(max_xor16(x)) : sum_xor32(sum_xor16(x));
    return x;
}

} // namespace

#endif
