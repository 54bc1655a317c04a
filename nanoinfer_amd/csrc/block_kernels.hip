// block_kernels.hip -- gfx950 kernels of the block-scaled cache (NI_KV_B8): e4m3
// values, one power-of-two scale for each (page, head) of K and of V.
//
//   block_append_kernel, block_append_row_kernel   f32 rows into the pages, scales
//                         grown where they must
//   block_attn_kernel     16 slots (query heads of rows that read the same cache
//                         head) over a run of keys, on the matrix cores
//   values_kernel         what the cache stands for, in f32 (any pool)
//
// A block's bytes lie in the order in which the lanes of block_attn_kernel take
// them to matrix products, so that a page needs no LDS on its way: lane l loads the
// 16 bytes at 16 l of each KB.  Of K they are dims 16 (l / 16) .. + 15 of
// position l % 16; of V positions 4 (l / 16) .. + 3 of dims l % 16 + 16 (0..3).
#include "kv_device.h"
#include "ops_plan.h"

namespace ni {
namespace {

constexpr float kTop = 448.f;  // the largest e4m3 value
constexpr int kMinExp = -117, kMaxExp = 120;

// Bytes of value (position p, dim d) within its block.
__device__ __forceinline__ uint32_t k_byte(uint32_t p, uint32_t d) {
    return d / 64 * 1024 + d % 64 / 16 * 256 + p * 16 + d % 16;
}
__device__ __forceinline__ uint32_t v_byte(uint32_t p, uint32_t d) {
    return d / 64 * 1024 + p / 4 * 256 + d % 16 * 16 + d % 64 / 16 * 4 + p % 4;
}

__device__ __forceinline__ float pow2(int e) { return __int_as_float((e + 127) << 23); }  // -126 <= e <= 127

// The exponent of the scale that values up to `top` (finite, not negative) need:
// top <= 448 * 2^e = 1.75 * 2^(e + 8).
__device__ __forceinline__ int scale_exp(float top) {
    const uint32_t b = __float_as_uint(top);
    const int e = (int)(b >> 23) - 127 - 8 + ((b & 0x7fffffu) > 0x600000u ? 1 : 0);
    return min(max(e, kMinExp), kMaxExp);
}
// The exponent of a stored scale; below every other where nothing was stored yet.
__device__ __forceinline__ int exp_of(float scale) { return (int)(__float_as_uint(scale) >> 23) - 127; }

__device__ __forceinline__ float wave_max(float x) {
    x = fmaxf(x, dpp_move<0xb1>(x));
    x = fmaxf(x, dpp_move<0x4e>(x));
    x = fmaxf(x, dpp_move<0x141>(x));
    x = fmaxf(x, dpp_move<0x140>(x));
    return rows4_max(x);
}

// The largest value that is stored with scale 2^e: of the largest scale's, 256 (which f32's
// largest would become) does not fit f32; 240 is half a step from it.
__device__ __forceinline__ float largest(int e) { return e == kMaxExp ? 240.f : kTop; }

// Four values times `inv` as e4m3, to nearest even, at most `most`.
__device__ __forceinline__ uint32_t e4m3x4(float a, float b, float c, float d, float inv, float most = kTop) {
    const auto in = [&](float x) { return fminf(fmaxf(x * inv, -most), most); };
    const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(in(a), in(b), 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(in(c), in(d), lo, true);
}
// Four stored values times `by` (a power of two, at most 1), rounded again.
__device__ __forceinline__ uint32_t rescale4(uint32_t w, float by) {
    const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
    return e4m3x4(lo[0], lo[1], hi[0], hi[1], by);
}
// An input as it is stored: a NaN as 0 (an infinity ends at the largest value).
__device__ __forceinline__ float number(float x) { return x == x ? x : 0.f; }
__device__ __forceinline__ float finite_size(float x) {
    const float y = fabsf(x);
    return y < INFINITY ? y : 0.f;
}

// One wave per (page of the call, layer, head) and K or V.  A lane holds the 16
// bytes that it loads in block_attn_kernel: of K a position's 16 dims (those of
// positions that are not new only where the scale grows), of V four positions
// of four dims, merged with what is there where not all of them are new.
// Bound by memory, from some thousand waves on (84 MB 21 us, 4.0 TB/s); of 2047 rows of 8 heads x
// 128, 21 MB in 2064 waves, 9.1 us, the launch's start and each wave's loads, maximum and stores,
// one after another, are half.
template <int D, int INL>
__global__ __launch_bounds__(256) void block_append_kernel(const BlockAppendLaunch a, const PlanArg<INL> pa) {
    constexpr int NB = D / 64;
    const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t H = a.pool.n_head;
    const uint64_t unit = (uint64_t)blockIdx.x * 4 + wave;  // ((entry, layer), head, K | V)
    const uint32_t is_v = (uint32_t)(unit & 1), head = (uint32_t)(unit / 2 % H);
    const uint32_t el = (uint32_t)(unit / 2 / H);
    if (el >= a.n * a.n_lay) return;
    const uint32_t entry = el / a.n_lay, lay = el - entry * a.n_lay;
    const uint8_t* plan = plan_base(pa, a.plan);
    const BlockAppend e = reinterpret_cast<const BlockAppend*>(plan)[entry];
    const uint32_t* list = reinterpret_cast<const uint32_t*>(plan + a.off_list);
    uint8_t* const page = reinterpret_cast<uint8_t*>(a.pool.k + (uint64_t)(a.layer0 + lay) * a.pool.layer_halves +
                                                     (uint64_t)e.page * a.pool.page_halves);
    uint8_t* const block = page + ((uint64_t)head * 2 + is_v) * kPage * D;
    float* const scale = reinterpret_cast<float*>(page + a.pool.b8) + 2 * head + is_v;
    const float before = *scale;
    const uint32_t slots = e.slots & 0xffffu;
    const float* const in = (is_v ? a.v : a.k) + (int64_t)lay * a.layer_stride + head * D;
    // Input row of position p; of one that is not new the first row, whose values are
    // dropped (loads that no branch parts are in flight together).
    auto row_of = [&](uint32_t p, bool mine) {
        const uint32_t i = e.src + (mine ? __popc(slots & ((1u << p) - 1u)) : 0);
        return (int64_t)(e.slots & kListed ? list[i] : i) * a.row_stride;
    };
    const uint32_t hi = lane >> 4, lo = lane & 15u;
    // What a lane's bytes hold beside new ones is asked for with the rows, not behind them.
    const uint32_t four = slots >> (4 * hi) & 15u;
    const bool beside = is_v && four != 0 && four != 15u;
    u32x4 held[NB];
#pragma unroll
    for (int i = 0; i < NB; i++) {
        held[i] = u32x4{0, 0, 0, 0};
        if (beside) held[i] = reinterpret_cast<const u32x4*>(block + 1024 * i)[lane];
    }
    // x[i][4 w + b]: the value of byte 4 w + b of the lane's 16 of run i
    float x[NB][16];
    bool mine[4];  // of V position 4 hi + b is new; of K all alike
    float top = 0.f;
    if (!is_v) {
#pragma unroll
        for (int b = 0; b < 4; b++) mine[b] = slots >> lo & 1;
        const float* p = in + row_of(lo, mine[0]) + 16 * hi;
#pragma unroll
        for (int i = 0; i < NB; i++)
#pragma unroll
            for (int w = 0; w < 4; w++) {
                const float4 y = *reinterpret_cast<const float4*>(p + 64 * i + 4 * w);
                x[i][4 * w] = y.x;
                x[i][4 * w + 1] = y.y;
                x[i][4 * w + 2] = y.z;
                x[i][4 * w + 3] = y.w;
            }
    } else {
#pragma unroll
        for (int b = 0; b < 4; b++) {
            mine[b] = slots >> (4 * hi + b) & 1;
            const float* p = in + row_of(4 * hi + b, mine[b]) + lo;
#pragma unroll
            for (int i = 0; i < NB; i++)
#pragma unroll
                for (int w = 0; w < 4; w++) x[i][4 * w + b] = p[64 * i + 16 * w];
        }
    }
#pragma unroll
    for (int i = 0; i < NB; i++)
#pragma unroll
        for (int j = 0; j < 16; j++) {
            x[i][j] = mine[j % 4] ? x[i][j] : 0.f;
            top = fmaxf(top, finite_size(x[i][j]));
            x[i][j] = number(x[i][j]);
        }
    top = wave_max(top);
    const bool anew = e.slots & kAnew;  // the block begins with this call, whatever its scale was
    const int old = exp_of(before), need = scale_exp(top), now = anew ? need : max(old, need);
    const float inv = pow2(-now), most = largest(now);
    // Old values that stay: by how much they shrink (nothing is there yet below kMinExp).
    const bool grown = !anew && now > old;
    const float by = old < kMinExp ? 0.f : pow2(max(old - now, -126));
    const bool any = mine[0] || mine[1] || mine[2] || mine[3], all = mine[0] && mine[1] && mine[2] && mine[3];
    if (any || grown) {
#pragma unroll
        for (int i = 0; i < NB; i++) {
            u32x4* at = reinterpret_cast<u32x4*>(block + 1024 * i) + lane;
            u32x4 y = held[i];
            if (!all && !beside) y = *at;
#pragma unroll
            for (int w = 0; w < 4; w++) {
                const uint32_t fresh = e4m3x4(x[i][4 * w], x[i][4 * w + 1], x[i][4 * w + 2], x[i][4 * w + 3], inv, most);
                const uint32_t kept = grown ? rescale4(y[w], by) : y[w];
                const uint32_t take = (mine[0] ? 0xffu : 0u) | (mine[1] ? 0xff00u : 0u) | (mine[2] ? 0xff0000u : 0u) |
                                      (mine[3] ? 0xff000000u : 0u);
                y[w] = (fresh & take) | (kept & ~take);
            }
            *at = y;
        }
    }
    if (lane == 0 && (anew || grown)) *scale = pow2(now);
}

// The same where every page takes one row, as in a decode step: 16 lanes per (page,
// layer, head) and K or V, 4 D / 64 dims of the row to a lane (with a wave each, whose
// lanes had little to do, 64 rows x 12 layers x 12 heads took 12.5 us, so 5.4; of one layer 3.6,
// a launch).  Of K a lane stores its own
// bytes, of V it merges them with the 16 that hold three other positions.  Where the scale
// grows the lanes go over the block, 16 bytes each in turn.
template <int D, int INL>
__global__ __launch_bounds__(256) void block_append_row_kernel(const BlockAppendLaunch a, const PlanArg<INL> pa) {
    constexpr int NB = D / 64;
    const uint32_t x16 = threadIdx.x & 15u;
    const uint32_t H = a.pool.n_head;
    const uint64_t unit = ((uint64_t)blockIdx.x * 256 + threadIdx.x) / 16;  // ((entry, layer), head, K | V)
    const uint32_t is_v = (uint32_t)(unit & 1), eh = (uint32_t)(unit / 2), el = eh / H, head = eh - el * H;
    if (el >= a.n * a.n_lay) return;
    const uint32_t entry = el / a.n_lay, lay = el - entry * a.n_lay;
    const uint8_t* plan = plan_base(pa, a.plan);
    const BlockAppend e = reinterpret_cast<const BlockAppend*>(plan)[entry];
    uint8_t* const page = reinterpret_cast<uint8_t*>(a.pool.k + (uint64_t)(a.layer0 + lay) * a.pool.layer_halves +
                                                     (uint64_t)e.page * a.pool.page_halves);
    uint8_t* const block = page + ((uint64_t)head * 2 + is_v) * kPage * D;
    float* const scale = reinterpret_cast<float*>(page + a.pool.b8) + 2 * head + is_v;
    const float before = *scale;
    const uint32_t slot = (uint32_t)__ffs(e.slots & 0xffffu) - 1u;
    const uint32_t src = e.slots & kListed ? reinterpret_cast<const uint32_t*>(plan + a.off_list)[e.src] : e.src;
    const float* const in = (is_v ? a.v : a.k) + (int64_t)lay * a.layer_stride + (int64_t)src * a.row_stride + head * D;
    // dim of value (i, w): 64 i + 4 x16 + w of K, 64 i + 16 w + x16 of V
    const float* const mine = in + (is_v ? x16 : 4 * x16);
    const uint32_t step = is_v ? 16 : 1;
    u32x4 held[NB];
    float x[NB][4], top = 0.f;
#pragma unroll
    for (int i = 0; i < NB; i++) {
        held[i] = reinterpret_cast<const u32x4*>(block + 1024 * i + slot / 4 * 256)[x16];  // (V: beside the new bytes)
#pragma unroll
        for (int w = 0; w < 4; w++) x[i][w] = mine[64 * i + step * w];
    }
#pragma unroll
    for (int i = 0; i < NB; i++)
#pragma unroll
        for (int w = 0; w < 4; w++) {
            top = fmaxf(top, finite_size(x[i][w]));
            x[i][w] = number(x[i][w]);
        }
    top = fmaxf(top, dpp_move<0xb1>(top));
    top = fmaxf(top, dpp_move<0x4e>(top));
    top = fmaxf(top, dpp_move<0x141>(top));
    top = fmaxf(top, dpp_move<0x140>(top));
    const bool anew = e.slots & kAnew;  // the block begins with this row, whatever its scale was
    const int old = exp_of(before), need = scale_exp(top), now = anew ? need : max(old, need);
    const float inv = pow2(-now), most = largest(now);
    const bool grown = !anew && now > old;
    const float by = old < kMinExp ? 0.f : pow2(max(old - now, -126));
#pragma unroll
    for (int i = 0; i < NB; i++) {
        u32x4* const words = reinterpret_cast<u32x4*>(block + 1024 * i);
        const uint32_t fresh = e4m3x4(x[i][0], x[i][1], x[i][2], x[i][3], inv, most);
        if (grown)
            for (uint32_t hi = 0; hi < 4; hi++) {
                if (is_v ? hi == slot / 4 : x16 == slot) continue;  // (K: the row itself)
                u32x4 y = words[16 * hi + x16];
#pragma unroll
                for (int w = 0; w < 4; w++) y[w] = rescale4(y[w], by);
                words[16 * hi + x16] = y;
            }
        if (is_v) {
            u32x4 y = held[i];
            const uint32_t at = 8 * (slot % 4);
#pragma unroll
            for (int w = 0; w < 4; w++) {
                if (grown) y[w] = rescale4(y[w], by);
                y[w] = (y[w] & ~(0xffu << at)) | (fresh >> (8 * w) & 0xffu) << at;
            }
            words[16 * (slot / 4) + x16] = y;
        } else {
            *reinterpret_cast<uint32_t*>(block + k_byte(slot, 64 * i + 4 * x16)) = fresh;
        }
    }
    if (x16 == 0 && (anew || grown)) *scale = pow2(now);
}

// Eight stored values as f16, exactly (e4m3 lies within f16).
__device__ __forceinline__ half8_t e4m3_f16x8(uint32_t a, uint32_t b) {
    const half2_t x0 = __builtin_bit_cast(half2_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, 1.f, false));
    const half2_t x1 = __builtin_bit_cast(half2_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, 1.f, true));
    const half2_t x2 = __builtin_bit_cast(half2_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b, 1.f, false));
    const half2_t x3 = __builtin_bit_cast(half2_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b, 1.f, true));
    return half8_t{x0[0], x0[1], x1[0], x1[1], x2[0], x2[1], x3[0], x3[1]};
}
__device__ __forceinline__ half4_t e4m3_f16x4(uint32_t a) {
    const half2_t x0 = __builtin_bit_cast(half2_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, 1.f, false));
    const half2_t x1 = __builtin_bit_cast(half2_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, 1.f, true));
    return half4_t{x0[0], x0[1], x1[0], x1[1]};
}

// Weights are exp2(score - reference), the reference the running maximum less
// kRefLog2, raised when a score passes it by kRefLog2 + kRefSlack: at most 2^15 in f16
// (as hi + lo), normal down to 2^-24 of the largest.
constexpr float kRefLog2 = 10.f, kRefSlack = 5.f, kRefUnscale = 1.f / 1024.f;
// Weights of a page whose value scale is 2^-k of the outputs' unit enter a product 2^k
// smaller up to this k: what that costs them lies 2^-32 below the page's largest.
constexpr int kNear = 6;
// Others are added with the outputs brought to their units, where these stay finite: weights
// below 2^15, values below 2^9, a million keys to a wave.  Smaller scales add nothing.
constexpr int kFar = 83;

// One (item, layer, head), NT tiles of 16 slots: S^T = K Q^T (16 keys x 16 slots; q
// in f16 hi + lo parts, keys as stored, their page's scale on the sums), the online
// softmax down its columns, O^T += V^T P^T of two pages, in units of a value scale.  Lane l
// holds slot l % 16 of each tile and keys, then dims, 4 (l / 16) .. + 3: S^T's registers
// are P^T's operand as they are.  The W waves take two pages each in turn, the next
// ones' loads issued before the products of these; their states are joined through
// LDS.
//   Bound by memory for one tile: 16 sequences of 32 k keys, 4 query heads to each of 8 cache
// heads x 128, 1.03 GB, 158 us, 6.5 TB/s; 64 rows of 1..767 keys, 12 layers x 12 heads x 64, 0.41 GB,
// 77 us, 5.3 TB/s (short items: a start and a join to each 2 to 24 turns).  Two tiles are bound by
// what their waves issue: a prompt of 2041 rows x 32 query heads on 8 x 128, 34 GFLOP (69 with hi
// + lo), 88 us, of which the matrix cores are busy 28 and vector
// instructions (some 155 of a wave for two tiles of a page, 32 of them conversions) issue for 34; 512 rows
// x 16 x 12 heads x 64, 12 layers, 400 us.
template <int D, int NT, int W, bool MANY, int INL>
__global__ __launch_bounds__(64 * W) void block_attn_kernel(const PrefixLaunch a, const PlanArg<INL> pa) {
    constexpr int NB = D / 64, PB = 2, NC = 4 * NB;  // runs of 64 dims; pages of an iteration; 16-dim chunks
    // MANY: the queries are held once for all waves, in LDS, as each lane's operands.
    constexpr bool kShared = MANY;
    __shared__ union Lds {
        float red[W][kSlotTile][D + 4];  // of a tile: m, l, -, -, o
        half8_t q[NT][NB][2][kShared ? 2 : 1][64];
        __device__ Lds() {}
    } lds;
    auto& red = lds.red;
    __shared__ float tops[kShared ? NT : 1][2 * NB][kSlotTile];  // the queries' largest values, by step
    const int lane = threadIdx.x & 63;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t H = a.pool.n_head, lh = a.n_lay * H;
    const uint8_t* plan = plan_base(pa, a.plan);
    const uint32_t item_i = blockIdx.x / lh;
    const uint32_t rem = blockIdx.x - item_i * lh;
    const uint32_t lay = rem / H, head = rem - lay * H;
    const PrefixItem it = reinterpret_cast<const PrefixItem*>(plan + a.off_items)[item_i];
    const int col = lane & 15, rg = lane >> 4;
    typedef const __attribute__((address_space(4))) uint32_t* Words;
    typedef const __attribute__((address_space(4))) float* Scales;
    const Words tab = (Words)(plan + a.off_table) + it.tab;
    const uint8_t* const layer = reinterpret_cast<const uint8_t*>(a.pool.k + (uint64_t)(a.layer0 + lay) * a.pool.layer_halves);
    const uint64_t page_bytes = 2 * a.pool.page_halves;
    const uint32_t at_block = head * 2 * kPage * D, at_scale = a.pool.b8 + 8 * head;
    const uint32_t pg_end = (it.kv_end + kPage - 1) / kPage;

    struct Regs {
        u32x4 k[PB][NB], v[PB][NB];
    };
    // (runs of many slots read each page many times, from the caches; others once)
    auto load16 = [](const u32x4* p) { return MANY ? *p : __builtin_nontemporal_load(p); };
    // (page ids are asked for a turn ahead of the pages: one that waited for its id would wait twice)
    auto pages = [&](uint32_t pg, uint32_t (&id)[PB]) {
#pragma unroll
        for (int b = 0; b < PB; b++) id[b] = tab[min(pg + b, pg_end - 1)];  // (past the end: the last again, its keys masked)
    };
    auto load = [&](const uint32_t (&id)[PB], Regs& r, bool k, bool v) {
#pragma unroll
        for (int b = 0; b < PB; b++) {
            const u32x4* p = reinterpret_cast<const u32x4*>(layer + id[b] * page_bytes + at_block) + lane;
#pragma unroll
            for (int i = 0; i < NB; i++)
                if (k) r.k[b][i] = load16(p + 64 * i);
#pragma unroll
            for (int i = 0; i < NB; i++)
                if (v) r.v[b][i] = load16(p + 64 * (NB + i));
        }
    };
    auto scales = [&](const uint32_t (&id)[PB], float (&ks)[PB], float (&vs)[PB]) {
#pragma unroll
        for (int b = 0; b < PB; b++) {
            const Scales sc = (Scales)(layer + id[b] * page_bytes + at_scale);
            ks[b] = sc[0];
            vs[b] = sc[1];
        }
    };
    Regs cur;
    uint32_t pg = it.kv_begin / kPage + wave * PB;
    uint32_t id[PB];  // of the next turn's pages
    float ks[PB], vs[PB];
    pages(pg, id);
    if (pg < pg_end) load(id, cur, true, true);
    scales(id, ks, vs);
    pages(pg + W * PB, id);

    const uint32_t first_pos = min(it.pos0 + it.slot0 / a.group, kWholePos);  // of the item's first slot
    const uint32_t plain_end = min(it.kv_end, first_pos + 1);                 // every slot sees the keys before it
    const uint32_t plain_pages = first_pos / kPage + 1;                       // and keys of each page before this
    uint32_t qend[NT];  // the slot sees the keys before it
    // A slot's query enters products with its largest value in 2^14 .. 2^15, the power of two that
    // takes on the keys' scales: keys may be of any size, and queries small or large to match.
    float qs[NT];
    half8_t qh[kShared ? 1 : NB][2], ql[kShared ? 1 : NB][2];
    // Shared: a wave brings step (wave / 2, wave % 2) of every tile, of one with 64 dims a step of one
    // (of a single tile two waves bring none).
    constexpr int STEPS = kShared ? 1 : 2 * NB;
    static_assert(!kShared || W == 4, "a step of every tile to a wave, or two");
    const int step0 = NB == 2 ? (int)wave : (int)wave % 2;
    auto brings = [&](int t) { return !kShared || NB == 2 || (int)wave / 2 == t; };
    float x[NT][STEPS][8], most[NT];
#pragma unroll
    for (int t = 0; t < NT; t++) {
        const bool has = t * (int)kSlotTile + col < (int)it.ns;
        const uint32_t slot = it.slot0 + (has ? t * kSlotTile + col : 0u);
        const uint32_t row = slot / a.group, g = slot - row * a.group;
        qend[t] = min(it.kv_end, min(it.pos0 + row, kWholePos) + 1);
        most[t] = 0.f;
        if (!brings(t)) continue;
        // step (i, j) of QK, number 2 i + j: dims 64 i + 16 rg + 8 j .. + 7, as the lane's bytes of K
        const float* qb = a.q + (int64_t)lay * a.q_layer_stride + (int64_t)(it.row0 + row) * a.q_row_stride +
                          (head * a.group + g) * D + 16 * rg;
#pragma unroll
        for (int i = 0; i < STEPS; i++) {
            const int step = kShared ? step0 : i;
            const float4* p = reinterpret_cast<const float4*>(qb + 64 * (step / 2) + 8 * (step % 2));
            const float4 x0 = p[0], x1 = p[1];
            const float y[8] = {x0.x, x0.y, x0.z, x0.w, x1.x, x1.y, x1.z, x1.w};
#pragma unroll
            for (int e = 0; e < 8; e++) {
                x[t][i][e] = has ? y[e] : 0.f;
                most[t] = fmaxf(most[t], fabsf(x[t][i][e]));
            }
        }
        most[t] = rows4_max(most[t]);
        if (kShared && rg == 0) tops[t][step0][col] = most[t];
    }
    if constexpr (kShared) __syncthreads();
#pragma unroll
    for (int t = 0; t < NT; t++) {
        if constexpr (kShared) {
#pragma unroll
            for (int i = 0; i < 2 * NB; i++) most[t] = fmaxf(most[t], tops[t][i][col]);
        }
        const int up = min(141 - (int)(__float_as_uint(most[t] * a.qscale) >> 23), 126);
        const float grow = pow2(up);
        qs[t] = pow2(-up);
        if (!brings(t)) continue;
#pragma unroll
        for (int i = 0; i < STEPS; i++) {
            float y[8];
#pragma unroll
            for (int e = 0; e < 8; e++) {
                y[e] = x[t][i][e] * a.qscale * grow;
                asm("" : "+v"(y[e]));  // the f32 products, as the split's residual sees them
            }
            half8_t hi, lo;
            split8(y, hi, lo);
            if constexpr (kShared) {
                lds.q[t][step0 / 2][step0 % 2][0][lane] = hi;
                lds.q[t][step0 / 2][step0 % 2][1][lane] = lo;
            } else {
                qh[i / 2][i % 2] = hi;
                ql[i / 2][i % 2] = lo;
            }
        }
    }
    if constexpr (kShared) __syncthreads();
    float mref[NT], lsum[NT];
    bool set[NT];  // the reference is a score's (alike in the four lanes of a slot)
    float4_t o[NT][NC];
#pragma unroll
    for (int t = 0; t < NT; t++) {
        mref[t] = lsum[t] = 0.f;
        set[t] = false;
#pragma unroll
        for (int c = 0; c < NC; c++) o[t][c] = float4_t{0.f, 0.f, 0.f, 0.f};
    }

    int unit = kMinExp - 1;  // log2 of the largest value scale so far
    int seen[NT];            // and of those that a slot sees
#pragma unroll
    for (int t = 0; t < NT; t++) seen[t] = unit;
    for (; pg < pg_end; pg += W * PB) {
        // One tile: the next pages' registers beside these.  Two leave no room for that: keys
        // follow the products that read the last ones, values likewise.
        constexpr bool kBeside = !MANY;
        const bool more = pg + W * PB < pg_end;
        Regs nxt;
        if (kBeside && more) load(id, nxt, true, true);
        if constexpr (kShared) asm volatile("" : : : "memory");  // (the queries stay in LDS: not kept from one turn to the next)
        float4_t st[NT][PB];
        // (products that add to one sum stand apart, here and below: each waits for the one before)
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
            for (int b = 0; b < PB; b++) st[t][b] = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < NB; i++)
#pragma unroll
            for (int j = 0; j < 2; j++) {
                half8_t kh[PB], q_hi[NT], q_lo[NT];
#pragma unroll
                for (int t = 0; t < NT; t++) {
                    if constexpr (kShared) {
                        q_hi[t] = lds.q[t][i][j][0][lane];
                        q_lo[t] = lds.q[t][i][j][1][lane];
                    } else {
                        q_hi[t] = qh[i][j];
                        q_lo[t] = ql[i][j];
                    }
                }
#pragma unroll
                for (int b = 0; b < PB; b++) kh[b] = e4m3_f16x8(cur.k[b][i][2 * j], cur.k[b][i][2 * j + 1]);
#pragma unroll
                for (int t = 0; t < NT; t++)
#pragma unroll
                    for (int b = 0; b < PB; b++)
                        st[t][b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kh[b], q_lo[t], st[t][b], 0, 0, 0);
#pragma unroll
                for (int t = 0; t < NT; t++)
#pragma unroll
                    for (int b = 0; b < PB; b++)
                        st[t][b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kh[b], q_hi[t], st[t][b], 0, 0, 0);
            }
        if (!kBeside && more) load(id, cur, true, false);
        float next_ks[PB], next_vs[PB];
        uint32_t next_id[PB];
        scales(id, next_ks, next_vs);
        pages(pg + 2 * W * PB, next_id);
        // Outputs are kept in units of the largest value scale so far, 2^unit: exact, as far as
        // f32 reaches.  The weights of pages whose scale is no more than 2^kNear smaller
        // are taken in those units too, and both pages enter one product.  What a slot does not
        // see leaves it as it is: the scale of a second page that not all slots see has no part in
        // how the first is taken, and a slot's outputs are raised to the scales that it sees (a
        // slot that does not see a page sees none behind it).
        const int e[PB] = {exp_of(vs[0]), exp_of(vs[1])};
        const bool mixed = pg + 1 >= plain_pages && pg + 1 < pg_end;
        const int u0 = max(unit, mixed ? e[0] : max(e[0], e[1]));
        const int units[PB] = {u0, max(u0, e[1])};
        int near_by[PB], far_by[PB];  // log2 of what weights shrink by, or outputs grow by meanwhile
#pragma unroll
        for (int b = 0; b < PB; b++) {
            const int below = units[b] - e[b];
            near_by[b] = below <= kNear ? below : 0;
            far_by[b] = below <= kNear ? 0 : min(below, kFar + 1);
        }
        const bool both = units[0] == units[1] && (far_by[0] | far_by[1]) == 0;
        half8_t wh[NT], wl[NT];
#pragma unroll
        for (int t = 0; t < NT; t++) {
            float s[PB][4];
#pragma unroll
            for (int b = 0; b < PB; b++) {
                const float ref = mref[t] + (float)near_by[b];
#pragma unroll
                for (int j = 0; j < 4; j++) s[b][j] = fmaf(st[t][b][j], ks[b] * qs[t], -ref);
            }
            if ((pg + PB) * kPage > plain_end) {
#pragma unroll
                for (int b = 0; b < PB; b++) {
                    const int seen_keys = (int)(qend[t] - (pg + b) * kPage) - 4 * rg;
#pragma unroll
                    for (int j = 0; j < 4; j++)
                        if (j >= seen_keys) s[b][j] = -INFINITY;
                }
            }
            float lm = s[0][0];
#pragma unroll
            for (int b = 0; b < PB; b++)
#pragma unroll
                for (int j = 0; j < 4; j++) lm = fmaxf(lm, s[b][j]);
            if (__any(lm > kRefLog2 + kRefSlack || !set[t])) {
                const float mx = rows4_max(lm) - kRefLog2;
                // The first finite maximum sets the reference, later ones only raise it (a slot's own, whatever the others have).
                const bool none = mx == -INFINITY;
                const float d = set[t] ? mx > kRefSlack ? mx : 0.f : none ? 0.f : mx;
                const float alpha = set[t] ? fast_exp2(-d) : 1.f;  // (nothing is summed yet)
                set[t] = set[t] || !none;
                if (__any(alpha != 1.f)) {
                    lsum[t] *= alpha;
#pragma unroll
                    for (int c = 0; c < NC; c++) o[t][c] *= alpha;
                }
                mref[t] += d;
#pragma unroll
                for (int b = 0; b < PB; b++)
#pragma unroll
                    for (int j = 0; j < 4; j++) s[b][j] -= d;
            }
            half4_t ph[PB], pl[PB];
#pragma unroll
            for (int b = 0; b < PB; b++) {
                float p[4];
#pragma unroll
                for (int j = 0; j < 4; j++) p[j] = fast_exp2(s[b][j]);
                lsum[t] += ((p[0] + p[1]) + (p[2] + p[3])) * pow2(near_by[b]);
                split4(p, ph[b], pl[b]);
            }
            wh[t] = __builtin_shufflevector(ph[0], ph[1], 0, 1, 2, 3, 4, 5, 6, 7);
            wl[t] = __builtin_shufflevector(pl[0], pl[1], 0, 1, 2, 3, 4, 5, 6, 7);
        }
        // Both pages at once, or one at a time, the outputs in its units meanwhile.  (One body for
        // both, which drops the other page's values: with one of its own for pages by themselves
        // the compiler kept the outputs twice, 220 registers and two waves to a SIMD in place of 158
        // and three: the prompt above 102 us.)
#pragma unroll 1
        for (int b = 0; b < (both ? 1 : PB); b++) {
            const int up = b ? units[1] : units[0], by = b ? far_by[1] : far_by[0];
            const uint32_t with0 = both || (b == 0 && by <= kFar) ? ~0u : 0u, with1 = both || (b == 1 && by <= kFar) ? ~0u : 0u;
            if (up > unit) {
#pragma unroll
                for (int t = 0; t < NT; t++) {
                    if ((pg + b) * kPage >= qend[t]) continue;
                    if (unit >= kMinExp) {  // (else nothing is summed yet)
                        // (scales lie up to 2^237 apart)
                        const float down = pow2(max(unit - up, -126)), rest = pow2(min(max(unit - up + 126, -126), 0));
#pragma unroll
                        for (int c = 0; c < NC; c++) o[t][c] = o[t][c] * down * rest;
                    }
                    seen[t] = up;
                }
                unit = up;
            }
            if (by) {
#pragma unroll
                for (int t = 0; t < NT; t++)
#pragma unroll
                    for (int c = 0; c < NC; c++) o[t][c] *= by <= kFar ? pow2(by) : 1.f;
            }
            constexpr int G = 4 / NT;  // chunks at a time
#pragma unroll
            for (int c0 = 0; c0 < NC; c0 += G) {
                half8_t v8[G];
#pragma unroll
                for (int g = 0; g < G; g++) {
                    const int i = (c0 + g) / 4, c = (c0 + g) % 4;
                    v8[g] = e4m3_f16x8(cur.v[0][i][c] & with0, cur.v[1][i][c] & with1);
                }
#pragma unroll
                for (int g = 0; g < G; g++)
#pragma unroll
                    for (int t = 0; t < NT; t++)
                        o[t][c0 + g] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v8[g], wl[t], o[t][c0 + g], 0, 0, 0);
#pragma unroll
                for (int g = 0; g < G; g++)
#pragma unroll
                    for (int t = 0; t < NT; t++)
                        o[t][c0 + g] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v8[g], wh[t], o[t][c0 + g], 0, 0, 0);
            }
            if (by) {
#pragma unroll
                for (int t = 0; t < NT; t++)
#pragma unroll
                    for (int c = 0; c < NC; c++) o[t][c] *= by <= kFar ? pow2(-by) : 1.f;
            }
        }
        if (kBeside && more) cur = nxt;
        if (!kBeside && more) load(id, cur, false, true);
#pragma unroll
        for (int b = 0; b < PB; b++) {
            ks[b] = next_ks[b];
            vs[b] = next_vs[b];
            id[b] = next_id[b];
        }
    }
    // The waves' states of a tile at a time, through LDS.
#pragma unroll
    for (int t = 0; t < NT; t++) {
        if (kShared || t) __syncthreads();  // (the queries, or the last tile's states, are read)
        const uint32_t first = t * kSlotTile;
        // (sums of values near f32's largest would pass it before they are divided by the weights':
        // both are kept 2^32 smaller, the reference 32 higher)
        const float lift = seen[t] > 64 ? 32.f : 0.f, unscale = seen[t] > 64 ? kRefUnscale * 0x1p-32f : kRefUnscale;
        const float l = rows4_sum(lsum[t]);
        if (first + col < it.ns) {
            if (rg == 0)
                *reinterpret_cast<float2*>(&red[wave][col][0]) = float2{set[t] ? mref[t] + (kRefLog2 + lift) : kMinScore, l * unscale};
#pragma unroll
            for (int c = 0; c < NC; c++)
                *reinterpret_cast<float4_t*>(&red[wave][col][4 + c * 16 + 4 * rg]) = o[t][c] * (unscale * pow2(max(seen[t], kMinExp)));
        }
        __syncthreads();
        const uint32_t slots = it.ns > first ? min(it.ns - first, kSlotTile) : 0u;
        for (uint32_t u = threadIdx.x; u < slots * (D / 4); u += 64 * W) {
            const uint32_t sl = u / (D / 4), d = u % (D / 4) * 4;
            float M = red[0][sl][0];
#pragma unroll
            for (int w = 1; w < W; w++) M = fmaxf(M, red[w][sl][0]);
            float L = 0.f;
            float4_t O = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int w = 0; w < W; w++) {
                const float wt = fast_exp2(red[w][sl][0] - M);
                L += red[w][sl][1] * wt;
                O += *reinterpret_cast<const float4_t*>(&red[w][sl][4 + d]) * wt;
            }
            const uint32_t slot = first + sl;
            if (it.part0 == kNoSlot) {
                const uint32_t r = (it.slot0 + slot) / a.group, gg = it.slot0 + slot - r * a.group;
                *reinterpret_cast<float4_t*>(a.out + (int64_t)lay * a.out_layer_stride +
                                             (int64_t)(it.row0 + r) * a.out_row_stride + (head * a.group + gg) * D + d) = O / L;
            } else {
                const uint64_t part = ((uint64_t)(it.part0 + slot) * a.n_lay + lay) * H + head;
                *reinterpret_cast<float4_t*>(a.part_o + part * D + d) = O;
                if (d == 0) *reinterpret_cast<float2*>(a.part_ml + 2 * part) = float2{M, L};
            }
        }
    }
}

// Bound by the launch and its stores: 2047 rows of 8 heads x 128, 21 MB, 8.3 us; 64 rows 3.7.
// A thread takes four dims of a row and head of K or V: dims d .. + 3, of a
// block-scaled V dims d, d + 16, d + 32, d + 48 (one word of four positions each).
template <int INL>
__global__ __launch_bounds__(256) void values_kernel(const ValuesLaunch a, const PlanArg<INL> pa) {
    const uint32_t D = a.pool.head_dim, quads = D / 4, per_row = 2 * a.pool.n_head * quads;
    const uint64_t gid = (uint64_t)blockIdx.x * 256u + threadIdx.x;
    const uint64_t lr = gid / per_row;
    if (lr >= (uint64_t)a.n_lay * a.n_rows) return;
    uint32_t u = (uint32_t)(gid - lr * per_row);
    const uint32_t lay = (uint32_t)(lr / a.n_rows), row = (uint32_t)(lr - (uint64_t)lay * a.n_rows);
    const uint32_t is_v = u / (a.pool.n_head * quads);
    u -= is_v * a.pool.n_head * quads;
    const uint32_t head = u / quads, x = u - head * quads;
    const uint32_t place = reinterpret_cast<const uint32_t*>(plan_base(pa, a.plan) + a.off_entries)[row], slot = place % kPage;
    const uint16_t* const page = a.pool.k + (uint64_t)(a.layer0 + lay) * a.pool.layer_halves +
                                 (uint64_t)(place / kPage) * a.pool.page_halves;
    float* const out = (is_v ? a.v_out : a.k_out) + (int64_t)lay * a.layer_stride + (int64_t)row * a.row_stride + head * D;
    float4 y;
    if (a.pool.b8) {
        const uint8_t* block = reinterpret_cast<const uint8_t*>(page) + (head * 2 + is_v) * kPage * D;
        const float scale = reinterpret_cast<const float*>(reinterpret_cast<const uint8_t*>(page) + a.pool.b8)[2 * head + is_v];
        if (!is_v) {
            const uint32_t w = *reinterpret_cast<const uint32_t*>(block + k_byte(slot, 4 * x));
            const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
            y = float4{lo[0] * scale, lo[1] * scale, hi[0] * scale, hi[1] * scale};
        } else {
            const uint32_t d = x / 16 * 64 + x % 16;
            const u32x4 w = *reinterpret_cast<const u32x4*>(block + (v_byte(slot, d) & ~15u));
            float z[4];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                z[i] = __builtin_amdgcn_cvt_f32_fp8((int)(w[i] >> (8 * (slot % 4))), 0) * scale;
                out[d + 16 * i] = z[i];
            }
            return;
        }
    } else {
        const uint16_t* block = page + (uint64_t)head * a.pool.head_halves + (is_v ? a.pool.head_halves / 2 : 0);
        if (a.pool.q8) {
            const uint8_t* b = reinterpret_cast<const uint8_t*>(block);
            const uint32_t w = *reinterpret_cast<const uint32_t*>(b + slot * D + 4 * x);
            const float scale = reinterpret_cast<const float*>(b + kPage * D)[slot];
            y = float4{i8f(w, 0) * scale, i8f(w, 1) * scale, i8f(w, 2) * scale, i8f(w, 3) * scale};
        } else {
            const half4_t h = *reinterpret_cast<const half4_t*>(block + slot * D + 4 * x);
            y = float4{(float)h[0], (float)h[1], (float)h[2], (float)h[3]};
        }
    }
    reinterpret_cast<float4*>(out)[x] = y;
}

}  // namespace

hipError_t launch_block_append(const BlockAppendLaunch& a, const void* ip, uint32_t ib, hipStream_t s,
                               const LaunchTiming& t) {
    const uint64_t units = (uint64_t)a.n * a.n_lay * a.pool.n_head * 2;
    if (units == 0) return hipSuccess;
    return with_plan(a, ip, ib, [&](auto pa) {
        constexpr int INL = sizeof(pa.b) > 4 ? (int)sizeof(pa.b) : 0;
        if (a.single) {
            if (a.pool.head_dim == 64) return go(block_append_row_kernel<64, INL>, (units + 15) / 16, 256, s, t, a, pa);
            if (a.pool.head_dim == 128) return go(block_append_row_kernel<128, INL>, (units + 15) / 16, 256, s, t, a, pa);
            return hipErrorInvalidValue;
        }
        if (a.pool.head_dim == 64) return go(block_append_kernel<64, INL>, (units + 3) / 4, 256, s, t, a, pa);
        if (a.pool.head_dim == 128) return go(block_append_kernel<128, INL>, (units + 3) / 4, 256, s, t, a, pa);
        return hipErrorInvalidValue;
    });
}

template <int D, int INL>
static hipError_t block_attn_t(const PrefixLaunch& a, uint64_t blocks, hipStream_t s, const LaunchTiming& t, const PlanArg<INL>& pa) {
    if (a.wide == 2) return go(block_attn_kernel<D, 2, 4, true, INL>, blocks, 256, s, t, a, pa);
    if (a.wide == 1) return go(block_attn_kernel<D, 1, 4, true, INL>, blocks, 256, s, t, a, pa);
    if (a.waves == 8) return go(block_attn_kernel<D, 1, 8, false, INL>, blocks, 512, s, t, a, pa);
    if (a.waves == 2) return go(block_attn_kernel<D, 1, 2, false, INL>, blocks, 128, s, t, a, pa);
    return go(block_attn_kernel<D, 1, 4, false, INL>, blocks, 256, s, t, a, pa);
}

hipError_t launch_block_attention(const PrefixLaunch& a, const void* ip, uint32_t ib, hipStream_t s,
                                  const LaunchTiming& t) {
    const uint64_t blocks = (uint64_t)a.n_items * a.n_lay * a.pool.n_head;
    if (blocks == 0) return hipSuccess;
    return with_plan(a, ip, ib, [&](auto pa) {
        constexpr int INL = sizeof(pa.b) > 4 ? (int)sizeof(pa.b) : 0;
        if (a.pool.head_dim == 64) return block_attn_t<64, INL>(a, blocks, s, t, pa);
        if (a.pool.head_dim == 128) return block_attn_t<128, INL>(a, blocks, s, t, pa);
        return hipErrorInvalidValue;
    });
}

hipError_t launch_gather_values(const ValuesLaunch& a, const void* ip, uint32_t ib, hipStream_t s) {
    const uint64_t threads = (uint64_t)a.n_lay * a.n_rows * 2 * a.pool.n_head * (a.pool.head_dim / 4);
    if (threads == 0) return hipSuccess;
    if (threads > 0xffffff00ull) return hipErrorInvalidValue;  // (handles allow 2^32 - 32)
    return with_plan(a, ip, ib, [&](auto pa) {
        constexpr int INL = sizeof(pa.b) > 4 ? (int)sizeof(pa.b) : 0;
        return go(values_kernel<INL>, (threads + 255) / 256, 256, s, {}, a, pa);
    });
}

}  // namespace ni
