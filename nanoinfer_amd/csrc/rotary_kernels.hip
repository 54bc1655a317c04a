// rotary_kernels.hip -- gfx950 kernels of the rotary positions.
//
//   rotary_kernel         rows of heads rotated to their positions
//   append_rotary_kernel  the cache append with keys rotated on their way into
//                         their pages and queries on their way out
//
// Pair i of a head turns by pos * f_i.  A frequency travels as its turns per
// position in 2^-64 units, within two of them, so pos * f_i modulo a turn is one
// 64-bit integer product, exact to pos * 2^-63 turns: no 64-bit floating point, and
// 2^-31 turns at most at any 32-bit position.
#include "kv_device.h"
#include "ops_plan.h"

namespace ni {
namespace {

// cos and sin of w * pos turns (w in 2^-64 turns a position), times scale.
// The turn fraction is reduced to an eighth either way of a quarter turn in
// integers, so the f32 angle is at most pi/4; its conversion, constant and product
// round it by up to 2^-24 of itself each.  The Taylor sums end below 2e-9 of the
// result there.
__device__ __forceinline__ void turn(uint64_t w, int64_t pos, float scale, float& c, float& s) {
    const uint64_t f = w * (uint64_t)pos;
    const uint32_t quarter = (uint32_t)((f + (1ull << 61)) >> 62);       // 0..3, to the nearest
    const int64_t rest = (int64_t)(f - ((uint64_t)quarter << 62));        // [-2^61, 2^61)
    const float x = (float)rest * 3.4061215800304394e-19f;                // 2 pi / 2^64
    const float z = x * x;
    const float ps = x + x * (z * (-1.f / 6 + z * (1.f / 120 + z * (-1.f / 5040 + z * (1.f / 362880)))));
    const float pc = 1.f + z * (-0.5f + z * (1.f / 24 + z * (-1.f / 720 + z * (1.f / 40320 - z * (1.f / 3628800)))));
    const float ss = (quarter & 1) ? pc : ps, cc = (quarter & 1) ? ps : pc;
    s = (quarter & 2) ? -ss * scale : ss * scale;
    c = (((quarter + 1) & 2) ? -cc : cc) * scale;
}

// Types of a row: four values from or to memory.
struct F32 {
    using T = float;
    static __device__ __forceinline__ float get(T x) { return x; }
    static __device__ __forceinline__ T put(float x) { return x; }
};
struct F16 {
    using T = _Float16;
    static __device__ __forceinline__ float get(T x) { return (float)x; }
    static __device__ __forceinline__ T put(float x) { return (T)x; }
};
struct BF16 {
    using T = __bf16;
    static __device__ __forceinline__ float get(T x) { return (float)x; }
    static __device__ __forceinline__ T put(float x) { return (T)x; }
};

template <typename E>
__device__ __forceinline__ float4 get4(const typename E::T* p) {
    typedef typename E::T V __attribute__((ext_vector_type(4)));
    const V v = *reinterpret_cast<const V*>(p);
    return float4{E::get(v[0]), E::get(v[1]), E::get(v[2]), E::get(v[3])};
}
template <typename E>
__device__ __forceinline__ void put4(typename E::T* p, const float4 x) {
    typedef typename E::T V __attribute__((ext_vector_type(4)));
    V v;
    v[0] = E::put(x.x);
    v[1] = E::put(x.y);
    v[2] = E::put(x.z);
    v[3] = E::put(x.w);
    *reinterpret_cast<V*>(p) = v;
}

// A chunk of 8 values of a head: pairs 4c .. 4c+3 below rot_dim (two runs of
// four values rot_dim/2 apart, or one run of eight when pairs are
// interleaved), values 8c .. 8c+7 past it.  lo and hi: where its two runs of
// four begin.
struct Chunk {
    uint32_t lo, hi;
    bool turned;
};
__device__ __forceinline__ Chunk chunk_of(uint32_t c, uint32_t rot_dim, uint32_t interleaved) {
    Chunk k;
    k.turned = 8 * c < rot_dim;
    const bool split = k.turned && !interleaved;
    k.lo = split ? 4 * c : 8 * c;
    k.hi = split ? rot_dim / 2 + 4 * c : 8 * c + 4;
    return k;
}
// The chunk's values turned: c and s belong to pairs 4c .. 4c+3.
__device__ __forceinline__ void turn_chunk(float4& a, float4& b, uint32_t interleaved, const float (&c)[4],
                                           const float (&s)[4]) {
    float x[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w}, y[8];
#pragma unroll
    for (int j = 0; j < 4; j++) {
        if (interleaved) {
            y[2 * j] = x[2 * j] * c[j] - x[2 * j + 1] * s[j];
            y[2 * j + 1] = x[2 * j + 1] * c[j] + x[2 * j] * s[j];
        } else {
            y[j] = x[j] * c[j] - x[4 + j] * s[j];
            y[4 + j] = x[4 + j] * c[j] + x[j] * s[j];
        }
    }
    a = float4{y[0], y[1], y[2], y[3]};
    b = float4{y[4], y[5], y[6], y[7]};
}

// a.wide (many rows; head_dim and rot_dim multiples of 8, rows 16-byte aligned): one
// thread per (row, chunk) and a.heads_per heads, whose cosines it computes once; neighbouring threads
// hold neighbouring chunks, so a wave moves whole heads.  Bound by memory: 4095 rows
// x 40 heads x 128 in bf16, 84 MB, 16.5 us (5.1 TB/s, a copy's rate).
template <typename E>
__global__ __launch_bounds__(256) void rotary_kernel(const RotaryLaunch a, const ni_rotary r) {
    const uint32_t chunks = r.head_dim >> 3;
    const uint32_t hb = (a.n_head + a.heads_per - 1) / a.heads_per;
    const uint64_t gid = (uint64_t)blockIdx.x * 256u + threadIdx.x;
    const uint64_t t = gid / chunks;
    const uint32_t c = (uint32_t)(gid - t * chunks);
    const uint32_t row = (uint32_t)(t / hb);
    const uint32_t h0 = (uint32_t)(t - (uint64_t)row * hb);
    if (row >= a.n_rows) return;
    const auto* x = static_cast<const typename E::T*>(a.x) + (int64_t)row * a.x_stride;
    auto* y = static_cast<typename E::T*>(a.out) + (int64_t)row * a.out_stride;
    const Chunk k = chunk_of(c, r.rot_dim, r.interleaved);
    float cs[4] = {1.f, 1.f, 1.f, 1.f}, sn[4] = {0.f, 0.f, 0.f, 0.f};
    if (k.turned) {
        const int64_t pos = a.positions ? (int64_t)a.positions[row] : (int64_t)a.pos0 + row;
#pragma unroll
        for (int j = 0; j < 4; j++) turn(r.turns[4 * c + j], pos, r.scale, cs[j], sn[j]);
    }
    for (uint32_t h = h0; h < a.n_head; h += hb) {
        const uint32_t d = h * r.head_dim;
        float4 u = get4<E>(x + d + k.lo), w = get4<E>(x + d + k.hi);
        if (k.turned) turn_chunk(u, w, r.interleaved, cs, sn);
        put4<E>(y + d + k.lo, u);
        put4<E>(y + d + k.hi, w);
    }
}

// Few rows, or any even head_dim, rot_dim and address: one thread per pair (or two
// values past rot_dim), value by value.  64 x 12 x 64 in f32 2.5 us, a launch.
template <typename E>
__global__ __launch_bounds__(256) void rotary_any_kernel(const RotaryLaunch a, const ni_rotary r) {
    const uint32_t pairs = r.head_dim >> 1, turned = r.rot_dim >> 1;
    const uint64_t gid = (uint64_t)blockIdx.x * 256u + threadIdx.x;
    const uint64_t t = gid / pairs;
    const uint32_t i = (uint32_t)(gid - t * pairs);
    const uint32_t row = (uint32_t)(t / a.n_head);
    const uint32_t h = (uint32_t)(t - (uint64_t)row * a.n_head);
    if (row >= a.n_rows) return;
    const bool split = i < turned && !r.interleaved;
    const uint32_t d0 = h * r.head_dim + (split ? i : 2 * i);
    const uint32_t d1 = split ? d0 + turned : d0 + 1;
    const auto* x = static_cast<const typename E::T*>(a.x) + (int64_t)row * a.x_stride;
    auto* y = static_cast<typename E::T*>(a.out) + (int64_t)row * a.out_stride;
    float u = E::get(x[d0]), w = E::get(x[d1]);
    if (i < turned) {
        const int64_t pos = a.positions ? (int64_t)a.positions[row] : (int64_t)a.pos0 + row;
        float c, s;
        turn(r.turns[i], pos, r.scale, c, s);
        const float p = u * c - w * s;
        w = w * c + u * s;
        u = p;
    }
    y[d0] = E::put(u);
    y[d1] = E::put(w);
}

// ------------------------------------------------------------------ append

// Eight values of one (position, head) of a Q8 pool, four at d0 and four at
// d1, held by a lane whose D/8 neighbours hold the rest (as q8_store8: scale
// = amax / 127, values rounded to nearest even).
__device__ __forceinline__ void q8_store4x2(uint8_t* blk, uint32_t D, uint32_t slot, uint32_t d0, uint32_t d1, bool first,
                                            const float4 x0, const float4 x1) {
    float a = fmaxf(fmaxf(fmaxf(fabsf(x0.x), fabsf(x0.y)), fmaxf(fabsf(x0.z), fabsf(x0.w))),
                    fmaxf(fmaxf(fabsf(x1.x), fabsf(x1.y)), fmaxf(fabsf(x1.z), fabsf(x1.w))));
    for (uint32_t off = 1; off < D / 8; off <<= 1) a = fmaxf(a, __shfl_xor(a, off));
    const float scale = a / 127.f;
    const float inv = scale > 0.f ? 1.f / scale : 0.f;
    uint8_t* row = blk + slot * D;
    *reinterpret_cast<uint32_t*>(row + d0) =
        q8_byte(x0.x, inv) | q8_byte(x0.y, inv) << 8 | q8_byte(x0.z, inv) << 16 | q8_byte(x0.w, inv) << 24;
    *reinterpret_cast<uint32_t*>(row + d1) =
        q8_byte(x1.x, inv) | q8_byte(x1.y, inv) << 8 | q8_byte(x1.z, inv) << 16 | q8_byte(x1.w, inv) << 24;
    if (first) reinterpret_cast<float*>(blk + kPage * D)[slot] = scale;
}

__device__ __forceinline__ uint2 pack4(const float4 a) {
    return uint2{f16_bits(a.x) | (f16_bits(a.y) << 16), f16_bits(a.z) | (f16_bits(a.w) << 16)};
}

// A workgroup takes one of a.parts shares of a (layer, row)'s chunks of q, k and v
// heads (in that order).  The row's cosines are computed once, by as many threads
// as there are pairs, while the chunks are on their way, and read back from LDS
// (each thread computing its own: 10.5 against 8.5 us for 12 layers x 160 rows x 36
// heads, 29.5 MB; 2047 rows x 48 heads x 128, 92 MB, 19.5 and 17.0, 5.4 TB/s).  The
// D/8 threads of a head are neighbours, aligned in the wave, and take the same
// branch: Q8 finds the head's largest value over them.
template <int INL>
__global__ __launch_bounds__(256) void append_rotary_kernel(const AppendRotaryLaunch a, const CacheRotary r,
                                                            const PlanArg<INL> pa) {
    constexpr int U = 4;  // chunks in flight
    __shared__ __attribute__((aligned(16))) float cs[kCachePairs], sn[kCachePairs];
    const uint32_t D = a.pool.head_dim, H = a.pool.n_head;
    const uint32_t shift = D == 64 ? 3 : 4;  // log2 of a head's chunks
    const uint32_t lr = blockIdx.x / a.parts, part = blockIdx.x - lr * a.parts;
    const uint32_t lay = lr / a.n_rows, row = lr - lay * a.n_rows;
    const uint32_t begin = part * a.share, end = min(begin + a.share, (a.n_q_head + 2 * H) << shift);
    const RotaryEntry e = reinterpret_cast<const RotaryEntry*>(plan_base(pa, a.plan) + a.off_entries)[row];
    const uint32_t page = e.place / kPage, slot = e.place % kPage;
    const float* q = a.q + (int64_t)lay * a.q_layer_stride + (int64_t)row * a.q_row_stride;
    float* q_out = a.q_out + (int64_t)lay * a.q_out_layer_stride + (int64_t)row * a.q_out_row_stride;
    const float* k = a.k + (int64_t)lay * a.layer_stride + (int64_t)row * a.row_stride;
    const float* v = a.v + (int64_t)lay * a.layer_stride + (int64_t)row * a.row_stride;
    const uint64_t block0 = (uint64_t)(a.layer0 + lay) * a.pool.layer_halves + (uint64_t)page * a.pool.page_halves;
    bool first = true;
    for (uint32_t t0 = begin + threadIdx.x; t0 - threadIdx.x < end; t0 += 256 * U) {
        float4 u[U], w[U];
#pragma unroll
        for (int j = 0; j < U; j++) {
            const uint32_t t = t0 + 256 * j;
            if (t >= end) continue;
            const uint32_t h = t >> shift;
            const bool is_v = h >= a.n_q_head + H;
            const Chunk c = chunk_of(t & ((1u << shift) - 1), is_v ? 0 : r.rot_dim, r.interleaved);
            const float* src = h < a.n_q_head ? q + h * D : is_v ? v + (h - a.n_q_head - H) * D : k + (h - a.n_q_head) * D;
            u[j] = get4<F32>(src + c.lo);
            w[j] = get4<F32>(src + c.hi);
        }
        if (first) {  // (the same for every thread)
            if (threadIdx.x < r.rot_dim / 2)
                turn(r.turns[threadIdx.x], (int64_t)e.pos, r.scale, cs[threadIdx.x], sn[threadIdx.x]);
            __syncthreads();
            first = false;
        }
#pragma unroll
        for (int j = 0; j < U; j++) {
            const uint32_t t = t0 + 256 * j;
            if (t >= end) continue;
            const uint32_t h = t >> shift, ci = t & ((1u << shift) - 1);
            const bool is_v = h >= a.n_q_head + H;
            const Chunk c = chunk_of(ci, is_v ? 0 : r.rot_dim, r.interleaved);
            if (c.turned) {
                const float4 c4 = *reinterpret_cast<const float4*>(cs + 4 * ci), s4 = *reinterpret_cast<const float4*>(sn + 4 * ci);
                const float cc[4] = {c4.x, c4.y, c4.z, c4.w}, ss[4] = {s4.x, s4.y, s4.z, s4.w};
                turn_chunk(u[j], w[j], r.interleaved, cc, ss);
            }
            if (h < a.n_q_head) {
                put4<F32>(q_out + h * D + c.lo, u[j]);
                put4<F32>(q_out + h * D + c.hi, w[j]);
                continue;
            }
            const uint64_t off = block0 + (uint64_t)(h - a.n_q_head - (is_v ? H : 0)) * a.pool.head_halves;
            if (a.pool.q8) {
                q8_store4x2(q8_block(a.pool, is_v, off), D, slot, c.lo, c.hi, ci == 0, u[j], w[j]);
            } else {
                uint16_t* dst = (is_v ? a.pool.v : a.pool.k) + off + slot * D;
                *reinterpret_cast<uint2*>(dst + c.lo) = pack4(u[j]);
                *reinterpret_cast<uint2*>(dst + c.hi) = pack4(w[j]);
            }
        }
    }
}

template <typename E>
hipError_t rotary_t(const RotaryLaunch& a, const ni_rotary& r, hipStream_t s) {
    if (a.wide) {
        const uint64_t hb = (a.n_head + a.heads_per - 1) / a.heads_per;
        const uint64_t threads = (uint64_t)a.n_rows * hb * (r.head_dim / 8);
        return go(rotary_kernel<E>, (threads + 255) / 256, 256, s, {}, a, r);
    }
    const uint64_t threads = (uint64_t)a.n_rows * a.n_head * (r.head_dim / 2);
    return go(rotary_any_kernel<E>, (threads + 255) / 256, 256, s, {}, a, r);
}

}  // namespace

hipError_t launch_rotary(const RotaryLaunch& a, const ni_rotary& r, hipStream_t s) {
    switch (a.dtype) {
        case NI_F32: return rotary_t<F32>(a, r, s);
        case NI_F16: return rotary_t<F16>(a, r, s);
        case NI_BF16: return rotary_t<BF16>(a, r, s);
        default: return hipErrorInvalidValue;
    }
}

hipError_t launch_append_rotary(const AppendRotaryLaunch& a, const CacheRotary& r, const void* ip, uint32_t ib,
                                hipStream_t s, const LaunchTiming& t) {
    const uint64_t blocks = (uint64_t)a.n_lay * a.n_rows * a.parts;
    if (blocks == 0) return hipSuccess;
    if (a.pool.head_dim != 64 && a.pool.head_dim != 128) return hipErrorInvalidValue;
    return with_plan(a, ip, ib, [&](auto pa) {
        constexpr int INL = sizeof(pa.b) > 4 ? (int)sizeof(pa.b) : 0;
        return go(append_rotary_kernel<INL>, blocks, 256, s, t, a, r, pa);
    });
}

}  // namespace ni
