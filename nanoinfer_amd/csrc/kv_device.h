// kv_device.h -- device helpers the gfx950 kernels share (kv_kernels.hip,
// rotary_kernels.hip, prefix_kernels.hip, verify_kernels.hip): vector types,
// f32 -> f16 and Q8 conversions, plans passed with the launch arguments, LDS
// tiles and DMA, and the launch helpers.
#pragma once

#include <hip/hip_ext.h>
#include <hip/hip_runtime.h>

#include <cstring>

#include "kv_plan.h"

namespace ni {
namespace {

typedef _Float16 half8_t __attribute__((ext_vector_type(8)));
typedef _Float16 half4_t __attribute__((ext_vector_type(4)));
typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
typedef float float4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// f32 -> f16 bits with round to nearest even (the hardware conversion under
// the default rounding mode keeps f16 subnormals and overflows to inf), NaN
// made canonical sign|0x7e00 -- the rules of crates/core/src/quant.rs:25-54.
__device__ __forceinline__ uint32_t f16_bits(float x) {
    uint32_t h = __builtin_bit_cast(uint16_t, static_cast<_Float16>(x));
    const uint32_t b = __float_as_uint(x);
    if ((b & 0x7fffffffu) > 0x7f800000u) h = ((b >> 16) & 0x8000u) | 0x7e00u;
    return h;
}

__device__ __forceinline__ uint4 pack8(const float4 a, const float4 b) {
    uint4 r;
    r.x = f16_bits(a.x) | (f16_bits(a.y) << 16);
    r.y = f16_bits(a.z) | (f16_bits(a.w) << 16);
    r.z = f16_bits(b.x) | (f16_bits(b.y) << 16);
    r.w = f16_bits(b.z) | (f16_bits(b.w) << 16);
    return r;
}

__device__ __forceinline__ float fast_exp2(float x) { return __builtin_amdgcn_exp2f(x); }

// Cross-lane move inside a row of 16 lanes (DPP; no LDS traffic).
template <int CTRL>
__device__ __forceinline__ float dpp_move(float v) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, false));
}

// Sum over the LPK consecutive lanes that hold one key row (LPK = 8 or 16).
template <int LPK>
__device__ __forceinline__ float key_sum(float x) {
    x += dpp_move<0xb1>(x);                            // quad_perm(1,0,3,2): lane ^ 1
    x += dpp_move<0x4e>(x);                            // quad_perm(2,3,0,1): lane ^ 2
    if constexpr (LPK >= 8) x += dpp_move<0x141>(x);   // row_half_mirror: the other quad of 8
    if constexpr (LPK >= 16) x += dpp_move<0x140>(x);  // row_mirror: the other 8 of 16
    return x;
}

// Running max starts at a finite sentinel so that exp2(m - m_new) of two
// empty states is 1 (not NaN); masked scores are -inf and weigh 0.
constexpr float kMinScore = -1e30f;

// A plan passed with the kernel arguments (N > 0) or left in device memory
// (N == 0: the launch struct's `plan` pointer).  Arguments live in the
// read-only kernarg segment; the kernels index it in place.
template <int N>
struct PlanArg {
    uint8_t b[N > 0 ? N : 4];
};

template <int N>
__device__ __forceinline__ const uint8_t* plan_base(const PlanArg<N>& pa, const uint8_t* dev) {
    if constexpr (N > 0)
        return pa.b;
    else
        return dev;
}

// A (page, head) block of a Q8 pool as bytes: [16][D] int8, then 16 scales.
__device__ __forceinline__ uint8_t* q8_block(const PoolGeom& pool, bool is_v, uint64_t off_halves) {
    return reinterpret_cast<uint8_t*>((is_v ? pool.v : pool.k) + off_halves);
}

__device__ __forceinline__ uint32_t q8_byte(float x, float inv) {
    return (uint32_t)(int32_t)fminf(fmaxf(rintf(x * inv), -127.f), 127.f) & 0xffu;
}

// Byte j of w as a signed integer, in f32.
__device__ __forceinline__ float i8f(uint32_t w, int j) { return (float)((int32_t)(w << (24 - 8 * j)) >> 24); }

// K/V loads are non-temporal: each byte is streamed once per step (156 -> 140
// us per config-3 launch against ordinary loads).
__device__ __forceinline__ u32x4 load16(const u32x4* p) { return __builtin_nontemporal_load(p); }

// Four signed int8 values (bytes 0..3 of w) as f16, exactly and bit for bit
// as static_cast<_Float16>: the f16 bit pattern 0x6400 | (b ^ 0x80) is 1024 +
// (b + 128), and subtracting 1152 leaves b (operands and result exactly
// representable, so the subtraction does not round).  Two values per byte
// permute (a byte to the low byte of each 16-bit half, zeros above), XOR and
// packed f16 subtract, against a bit extract and two conversions per value.
__device__ __forceinline__ half4_t i8x4_f16(uint32_t w) {
    const uint32_t lo = __builtin_amdgcn_perm(w, w, 0x0c010c00u) ^ 0x64806480u;  // bytes 0, 1
    const uint32_t hi = __builtin_amdgcn_perm(w, w, 0x0c030c02u) ^ 0x64806480u;  // bytes 2, 3
    const half2_t k1152 = {static_cast<_Float16>(1152.f), static_cast<_Float16>(1152.f)};
    const half2_t a = __builtin_bit_cast(half2_t, lo) - k1152;
    const half2_t b = __builtin_bit_cast(half2_t, hi) - k1152;
    return half4_t{a[0], a[1], b[0], b[1]};
}

// The hi + lo split of two softmax weights already scaled up (x in [0,
// 2^15]), packed: hi = f16(x), lo = f16(x - hi) unscaled, ~2^-22 relative
// where lo is normal and within 2^-25 absolute where it is subnormal.  One
// packed convert and one mixed-precision FMA per weight (x * 1 - hi, hi
// read as the f16 half of the packed register) instead of convert, convert
// back, subtract and convert; the same bits (checked on gfx950 against the
// plain formula over 2^21 pairs from 2^-40 to 2^16, zeros included).
__device__ __forceinline__ void split_w16x2(float x0, float x1, uint32_t& hi, uint32_t& lo) {
    const half2_t h = {static_cast<_Float16>(x0), static_cast<_Float16>(x1)};
    hi = __builtin_bit_cast(uint32_t, h);
    asm("v_fma_mixlo_f16 %0, %1, 1.0, -%2 op_sel_hi:[0,0,1]" : "=v"(lo) : "v"(x0), "v"(hi));
    asm("v_fma_mixhi_f16 %0, %1, 1.0, -%2 op_sel:[0,0,1] op_sel_hi:[0,0,1]" : "+v"(lo) : "v"(x1), "v"(hi));
}

// A matrix product may read what a vector instruction wrote two wait states ago
// at the earliest.  The compiler sees to that for instructions of its own, not
// for split_w16x2's: operands that go from there into a product pass through here
// (split4 and split8 see to it themselves).
__device__ __forceinline__ void settle(half4_t& a, half4_t& b) { asm("s_nop 1" : "+v"(a), "+v"(b)); }
__device__ __forceinline__ void settle(half8_t& a, half8_t& b) { asm("s_nop 1" : "+v"(a), "+v"(b)); }
__device__ __forceinline__ void settle(u32x4& a, u32x4& b, u32x4& c, u32x4& d) {
    asm("s_nop 1" : "+v"(a), "+v"(b), "+v"(c), "+v"(d));
}

// Four or eight values as operands of matrix products, hi and lo parts.
__device__ __forceinline__ void split4(const float (&x)[4], half4_t& hi, half4_t& lo) {
    uint32_t h0, l0, h1, l1;
    split_w16x2(x[0], x[1], h0, l0);
    split_w16x2(x[2], x[3], h1, l1);
    hi = __builtin_bit_cast(half4_t, u32x2_t{h0, h1});
    lo = __builtin_bit_cast(half4_t, u32x2_t{l0, l1});
    settle(hi, lo);
}
__device__ __forceinline__ void split8(const float (&x)[8], half8_t& hi, half8_t& lo) {
    u32x4 h, l;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        uint32_t hp, lp;
        split_w16x2(x[2 * i], x[2 * i + 1], hp, lp);
        h[i] = hp;
        l[i] = lp;
    }
    hi = __builtin_bit_cast(half8_t, h);
    lo = __builtin_bit_cast(half8_t, l);
    settle(hi, lo);
}

// Max and sum over lanes l, l ^ 16, l ^ 32, l ^ 48 (the four lanes holding
// one query column of an MFMA 16x16 output): v_permlane16_swap and
// v_permlane32_swap of a value with itself leave the two halves of each
// lane pair in the two results, so combining them is the pair's max or sum
// in both lanes.  No LDS round trip; the same bits as __shfl_xor.
__device__ __forceinline__ float rows4_max(float v) {
    u32x2_t s = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(s[0]), __uint_as_float(s[1]));
    s = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(s[0]), __uint_as_float(s[1]));
}

__device__ __forceinline__ float rows4_sum(float v) {
    u32x2_t s = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(s[0]) + __uint_as_float(s[1]);
    s = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(s[0]) + __uint_as_float(s[1]);
}

// Position, in 16-byte chunks, of chunk q of row `key` in an LDS tile of
// CH-chunk rows: row major, the chunk index XORed with a permutation of the
// row's 256-byte window index, so that the 16 lanes reading one chunk of 16
// consecutive rows (the K operand) and the 32 lanes reading 4 dims of 8 rows
// for the transposed V operand each hit distinct banks.
template <int CH>
__device__ __forceinline__ uint32_t tile_chunk(uint32_t key, uint32_t q) {
    const uint32_t i = (key * CH / 16) % CH;
    const uint32_t sw = ((i & (CH / 2 - 1)) << 1) | (i / (CH / 2));
    return key * CH + (q ^ sw);
}

typedef __fp16 v4fp16_t __attribute__((__vector_size__(4 * sizeof(__fp16))));

#define NI_LDS(p) ((__attribute__((address_space(3))) void*)(p))

// 16 bytes per lane from g to LDS at the wave-uniform dst + 16 * lane
// (global_load_lds_dwordx4, M0 = dst's LDS address).  Written as assembly
// so that the compiler does not add a wait for every DMA in flight before
// each LDS read it cannot prove disjoint from them: the caller waits
// (vmcnt) and synchronises itself.  The "memory" clobber and dst as an
// operand tell the compiler that LDS may change here.  The s_nop is the one
// wait state CDNA requires between a scalar write of M0 and an LDS-DMA load
// reading it; the compiler inserts it for its own code but cannot see into
// the asm.
__device__ __forceinline__ void lds_dma16(const void* g, void* dst) {
    const uint32_t m0 = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)NI_LDS(dst));
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" : : "v"(g), "s"(m0) : "memory", "m0");
}

// The same from a wave-uniform base plus a per-lane 32-bit byte offset (the
// SADDR form: no 64-bit address per lane), to the LDS byte address lds.
__device__ __forceinline__ void lds_dma16_sbase(const void* base, uint32_t off, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" : : "v"(off), "s"(base), "s"(lds)
                 : "memory", "m0");
}

// One kernel launch; with timing events the dispatch packet itself records
// the kernel's start and end (no separate event commands in the stream).
template <typename K, typename... Args>
hipError_t go(K kern, uint64_t blocks, uint32_t threads, hipStream_t s, const LaunchTiming& t, const Args&... args) {
    hipExtLaunchKernelGGL(kern, dim3((uint32_t)blocks), dim3(threads), 0, s, t.start, t.stop, 0, args...);
    return hipGetLastError();
}

// Launch `kern<INL>` with the plan inline (kInlinePlanTiny, kInlinePlanSmall
// or kInlinePlanBytes of arguments, the smallest that holds it) or through the
// device pointer in the launch struct.
template <typename L, typename Fn>
hipError_t with_plan(const L& a, const void* inline_plan, uint32_t inline_bytes, Fn&& launch) {
    if (inline_plan) {
        if (inline_bytes > kInlinePlanBytes) return hipErrorInvalidValue;
        if (inline_bytes <= kInlinePlanTiny) {
            PlanArg<kInlinePlanTiny> pa;
            memcpy(pa.b, inline_plan, inline_bytes);
            return launch(pa);
        }
        if (inline_bytes <= kInlinePlanSmall) {
            PlanArg<kInlinePlanSmall> pa;
            memcpy(pa.b, inline_plan, inline_bytes);
            return launch(pa);
        }
        PlanArg<kInlinePlanBytes> pa;
        memcpy(pa.b, inline_plan, inline_bytes);
        return launch(pa);
    }
    return launch(PlanArg<0>{});
}

}  // namespace
}  // namespace ni
