// prefix_kernels.hip -- gfx950 kernels of attention behind shared prefixes
// (ni_kv_prefix_attention): every row attends to the keys of its group's
// prefix, held once in the cache, and to its own sequence's.
//
//   prefix_attn_kernel   16 slots (query heads of rows that read the same
//                        cache head) over a run of keys; of a sequence's own
//                        keys it joins the prefix's partials and writes out
//   prefix_rows_kernel   the same for one or two slots of one row
//   prefix_wide_kernel   up to 128 slots over a run of a prefix's keys
//   prefix_merge_kernel  each slot's partial softmax states joined, where a
//                        sequence's own keys are partitioned too
//
// A prefix's keys leave memory once per 16 to 128 slots instead of once per
// row, and each product of the matrix cores serves all of them.
#include <type_traits>

#include "kv_device.h"
#include "ops_plan.h"

namespace ni {
namespace {

constexpr int kItemWaves = 4;        // waves of an item's workgroup
constexpr int kMergeWaves = 4;       // slots a merge workgroup joins
constexpr float kPScale = 16384.f;   // weights enter PV times 2^14: down to 4e-9 they are normal f16
constexpr float kPUnscale = 1.f / kPScale;
// Q8: where the value scales' reference starts.  Scales below it (values below
// 1e-28) lose bits; its inverse and its products with the unscalings are normal.
constexpr float kMinScale = 0x1p-100f;

// The power of two at or above x (0 of 0): the reference of scales up to x, which those
// of the pages to come seldom pass, and whose divisions are exact.
__device__ __forceinline__ float scale_reference(float x) {
    return __uint_as_float((__float_as_uint(x) + 0x7fffffu) & 0x7f800000u);
}

// One (item, layer, head): S^T = K Q^T (16 keys x 16 slots; q in f16 hi + lo
// parts), the online softmax down its columns, O^T += V^T P^T (p in hi + lo
// parts).  Lane l holds slot l % 16 and keys, then dims, 4 (l / 16) .. + 3.
// Pages go to LDS row major and come back as operands, V through the
// transposing read.  The W waves take every W-th page each; their states are joined
// through LDS, four dims of a slot to a thread.  For an item that writes out the
// thread joins the prefix's partials of its dims first, eight loads at a time,
// which arrive while the first pages do, and holds the sum to the end.  Bound by
// memory on long prefixes (16 rows x 32 heads x 128 behind 32767 keys, 595 MB with the
// rows' own keys: 90 us, 6.6 TB/s); on the Q8 cache by what a page costs a wave, which
// is paid once per 16 slots (~250 vector instructions, the f16 page's way into LDS), and by
// CUs with four workgroups where the mean is 3.4 (32 x 5 rows x 12 heads x 64 behind 2001:
// 12.7 us, 5.7 of them vector issue); by the start and the chain of pages of its
// longest items otherwise (48 rows x 32 query heads on 8 x 128, 1..511 own keys: 15 us).
template <int D, int INL, bool Q8>
__global__ __launch_bounds__(64 * kItemWaves) void prefix_attn_kernel(const PrefixLaunch a, const PlanArg<INL> pa) {
    constexpr int W = kItemWaves;
    constexpr int QC = D / 32;       // 32-dim chunks of QK
    constexpr int VC = D / 16;       // 16-dim chunks of PV
    constexpr int CH = D / 8;        // 16-byte chunks of an f16 row
    constexpr int LD = Q8 ? D / 64 : D / 32;  // 16-byte loads a lane makes of a page's K, and of its V
    constexpr size_t kTile = (size_t)kPage * D * 2;
    constexpr size_t kRed = (size_t)W * kSlotTile * (D + 4) * 4;
    constexpr size_t kLds = 2 * W * kTile > kRed ? 2 * W * kTile : kRed;
    __shared__ __attribute__((aligned(16))) uint8_t lds[kLds];
    auto& red = *reinterpret_cast<float(*)[W][kSlotTile][D + 4]>(lds);  // m, l, -, -, o

    const int lane = threadIdx.x & 63;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t H = a.pool.n_head, lh = a.n_lay * H;
    const uint8_t* plan = plan_base(pa, a.plan);
    const uint32_t item_i = blockIdx.x / lh;
    const uint32_t rem = blockIdx.x - item_i * lh;
    const uint32_t lay = rem / H, head = rem - lay * H;
    const PrefixItem it = reinterpret_cast<const PrefixItem*>(plan + a.off_items)[item_i];
    const int col = lane & 15, rg = lane >> 4;
    _Float16* const kt = reinterpret_cast<_Float16*>(lds + wave * 2 * kTile);
    _Float16* const vt = kt + kPage * D;

    const uint64_t off = (uint64_t)(a.layer0 + lay) * a.pool.layer_halves + (uint64_t)head * a.pool.head_halves;
    const uint32_t* __restrict__ tab = reinterpret_cast<const uint32_t*>(plan + a.off_table) + it.tab;
    const uint32_t pg_end = (it.kv_end + kPage - 1) / kPage;

    struct Regs {
        u32x4 k[LD], v[LD];
        float4 ks, vs;  // Q8: the scales of keys 4 rg .. + 3
    };
    auto load = [&](uint32_t pg, Regs& r) {
        const uint64_t at = off + (uint64_t)tab[pg] * a.pool.page_halves;
        const u32x4* kp = reinterpret_cast<const u32x4*>(a.pool.k + at) + lane;
        const u32x4* vp = reinterpret_cast<const u32x4*>(a.pool.v + at) + lane;
#pragma unroll
        for (int i = 0; i < LD; i++) r.k[i] = load16(kp + 64 * i);
#pragma unroll
        for (int i = 0; i < LD; i++) r.v[i] = load16(vp + 64 * i);
        if constexpr (Q8) {
            r.ks = *reinterpret_cast<const float4*>(q8_block(a.pool, false, at) + kPage * D + 16 * rg);
            r.vs = *reinterpret_cast<const float4*>(q8_block(a.pool, true, at) + kPage * D + 16 * rg);
        }
    };
    Regs cur;
    uint32_t pg = it.kv_begin / kPage + wave;
    if (pg < pg_end) load(pg, cur);

    const bool has = col < (int)it.ns;
    const uint32_t slot = it.slot0 + (has ? (uint32_t)col : 0u);
    const uint32_t row = slot / a.group, g = slot - row * a.group;
    const uint32_t qpos = min(it.pos0 + row, kWholePos);
    const uint32_t first_pos = min(it.pos0 + it.slot0 / a.group, kWholePos);  // of the item's first slot
    half8_t qh[QC], ql[QC];
    {
        const float* qb = a.q + (int64_t)lay * a.q_layer_stride + (int64_t)(it.row0 + row) * a.q_row_stride +
                          (head * a.group + g) * D + 8 * rg;
#pragma unroll
        for (int c = 0; c < QC; c++) {
            const float4 x0 = reinterpret_cast<const float4*>(qb + c * 32)[0];
            const float4 x1 = reinterpret_cast<const float4*>(qb + c * 32)[1];
            const float x[8] = {x0.x, x0.y, x0.z, x0.w, x1.x, x1.y, x1.z, x1.w};
            float y[8];
#pragma unroll
            for (int e = 0; e < 8; e++) {
                y[e] = has ? x[e] * a.qscale : 0.f;
                asm("" : "+v"(y[e]));  // the f32 products, as the split's residual sees them
            }
            split8(y, qh[c], ql[c]);
        }
    }
    float m = kMinScore, lsum = 0.f;
    float4_t o[VC];
#pragma unroll
    for (int c = 0; c < VC; c++) o[c] = float4_t{0.f, 0.f, 0.f, 0.f};
    constexpr int PG = kSlotTile * D / 4 / (64 * W);  // (slot, four dims) of a thread
    float pm[PG], pl[PG];
    float4_t po[PG];
#pragma unroll
    for (int g = 0; g < PG; g++) {
        const uint32_t t = threadIdx.x + 64 * W * g, sl = t / (D / 4), d = t % (D / 4) * 4;
        pm[g] = kMinScore;
        pl[g] = 0.f;
        po[g] = float4_t{0.f, 0.f, 0.f, 0.f};
        if (it.part0 != kNoSlot || sl >= it.ns) continue;
        constexpr uint32_t N = 8;
        for (uint32_t j0 = 0; j0 < it.n_pre; j0 += N) {
            float2 ml[N];
            float4_t x[N];
#pragma unroll
            for (uint32_t i = 0; i < N; i++) {  // (past the last: the last again, of no weight)
                const uint64_t part = ((uint64_t)(it.pre0 + sl + min(j0 + i, it.n_pre - 1) * it.pre_stride) * a.n_lay + lay) * H + head;
                ml[i] = *reinterpret_cast<const float2*>(a.part_ml + 2 * part);
                x[i] = *reinterpret_cast<const float4_t*>(a.part_o + part * D + d);
            }
            float mn = pm[g];
#pragma unroll
            for (uint32_t i = 0; i < N; i++) mn = fmaxf(mn, ml[i].x);
            const float keep = fast_exp2(pm[g] - mn);
            pm[g] = mn;
            pl[g] *= keep;
            po[g] *= keep;
#pragma unroll
            for (uint32_t i = 0; i < N; i++) {
                const float w = j0 + i < it.n_pre ? fast_exp2(ml[i].x - mn) : 0.f;
                pl[g] += ml[i].y * w;
                po[g] += x[i] * w;
            }
        }
    }
    // Q8: weights enter PV times scale / vref, at most 1: vref follows the largest
    // value scale that the slot has seen, so that the products keep the weights' bits
    // whatever the values' size.
    float vref = Q8 ? kMinScale : 1.f, vinv = 1.f / vref;

    for (; pg < pg_end; pg += W) {
        Regs nxt;
        if (pg + W < pg_end) load(pg + W, nxt);
        // Rows past kv_end enter as zeros: whatever the page holds there may
        // not reach a product, not even with weight 0.
#pragma unroll
        for (int i = 0; i < LD; i++) {
            if constexpr (Q8) {  // 16 values: chunks 2q, 2q + 1 of the row
                const uint32_t key = i * (1024 / D) + lane / (D / 16), q = 2 * (lane % (D / 16));
                const bool in = pg * kPage + key < it.kv_end;
                const u32x4 kq = in ? cur.k[i] : u32x4{0, 0, 0, 0}, vq = in ? cur.v[i] : u32x4{0, 0, 0, 0};
#pragma unroll
                for (int x = 0; x < 2; x++) {
                    *reinterpret_cast<half8_t*>(kt + tile_chunk<CH>(key, q + x) * 8) =
                        __builtin_shufflevector(i8x4_f16(kq[2 * x]), i8x4_f16(kq[2 * x + 1]), 0, 1, 2, 3, 4, 5, 6, 7);
                    *reinterpret_cast<half8_t*>(vt + tile_chunk<CH>(key, q + x) * 8) =
                        __builtin_shufflevector(i8x4_f16(vq[2 * x]), i8x4_f16(vq[2 * x + 1]), 0, 1, 2, 3, 4, 5, 6, 7);
                }
            } else {
                const uint32_t key = i * (512 / D) + lane / CH, q = lane % CH;
                const bool in = pg * kPage + key < it.kv_end;
                *reinterpret_cast<u32x4*>(kt + tile_chunk<CH>(key, q) * 8) = in ? cur.k[i] : u32x4{0, 0, 0, 0};
                *reinterpret_cast<u32x4*>(vt + tile_chunk<CH>(key, q) * 8) = in ? cur.v[i] : u32x4{0, 0, 0, 0};
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        // An infinity or NaN among the values that only the later of the item's
        // rows see: 0 times it would reach the earlier rows.
        bool stray = false;
        if constexpr (!Q8) {
            if (pg * kPage + kPage - 1 > first_pos) {
                uint32_t top = 0;
#pragma unroll
                for (int i = 0; i < LD; i++) {
                    const uint32_t key = pg * kPage + i * (512 / D) + lane / CH;
                    if (key > first_pos && key < it.kv_end) {
#pragma unroll
                        for (int w = 0; w < 4; w++)
                            top |= (uint32_t)((cur.v[i][w] & 0x7c00u) == 0x7c00u) |
                                   (uint32_t)((cur.v[i][w] & 0x7c000000u) == 0x7c000000u);
                    }
                }
                stray = __any(top != 0);
            }
        }
        float4_t st = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < QC; c++) {
            const half8_t kh = *reinterpret_cast<const half8_t*>(kt + tile_chunk<CH>(col, 4 * c + rg) * 8);
            st = __builtin_amdgcn_mfma_f32_16x16x32_f16(kh, ql[c], st, 0, 0, 0);
            st = __builtin_amdgcn_mfma_f32_16x16x32_f16(kh, qh[c], st, 0, 0, 0);
        }
        float s[4], mx = -INFINITY;
        bool seen[4];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const uint32_t key = pg * kPage + 4 * rg + j;
            seen[j] = key < it.kv_end && key <= qpos;
            float x = st[j];
            if constexpr (Q8) x *= cur.ks[j];
            s[j] = seen[j] ? x : -INFINITY;
            mx = fmaxf(mx, s[j]);
        }
        mx = rows4_max(mx);
        const float mn = fmaxf(m, mx);
        const float alpha = fast_exp2(m - mn);
        float oalpha = alpha;
        m = mn;
        float vs[4];
        if constexpr (Q8) {
            // Scales of keys that the lane's slot sees, each slot by itself: an
            // infinite or huge one of a later row may not reach the earlier ones.
            float vm = 0.f;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                vs[j] = seen[j] ? cur.vs[j] : 0.f;
                vm = fmaxf(vm, vs[j]);
            }
            if (__any(vm > vref)) {
                vm = fmaxf(scale_reference(rows4_max(vm)), vref);
                oalpha *= vref / vm;
                vref = vm;
                vinv = 1.f / vm;
            }
        }
        float p[4];
#pragma unroll
        for (int j = 0; j < 4; j++) p[j] = fast_exp2(s[j] - mn) * kPScale;
        lsum = lsum * alpha + ((p[0] + p[1]) + (p[2] + p[3]));
        if constexpr (Q8) {
#pragma unroll
            for (int j = 0; j < 4; j++) p[j] *= vs[j] * vinv;
        }
        half4_t ph, pl;
        split4(p, ph, pl);
        if (__any(oalpha != 1.f)) {
#pragma unroll
            for (int c = 0; c < VC; c++) o[c] *= oalpha;
        }
        auto pv = [&](int c, float4_t acc) {
            const int t = (lane >> 2) & 3, av = lane & 3;
            const _Float16* vp = vt + tile_chunk<CH>(4 * rg + t, 2 * c + (av >> 1)) * 8 + (av & 1) * 4;
            const half4_t v4 = __builtin_bit_cast(
                half4_t, __builtin_amdgcn_ds_read_tr16_b64_v4f16((__attribute__((address_space(3))) v4fp16_t*)(vp)));
            acc = __builtin_amdgcn_mfma_f32_16x16x16f16(v4, pl, acc, 0, 0, 0);
            return __builtin_amdgcn_mfma_f32_16x16x16f16(v4, ph, acc, 0, 0, 0);
        };
        if (!stray) {
#pragma unroll
            for (int c = 0; c < VC; c++) o[c] = pv(c, o[c]);
        } else {
            // Row by row, each with the values past its position as zeros, the
            // sums kept by the row's own slots alone.
            for (uint32_t r = it.slot0 / a.group; r <= (it.slot0 + it.ns - 1) / a.group; r++) {
#pragma unroll
                for (int i = 0; i < LD; i++) {
                    const uint32_t key = i * (512 / D) + lane / CH, q = lane % CH;
                    const bool in = pg * kPage + key < it.kv_end && pg * kPage + key <= it.pos0 + r;
                    *reinterpret_cast<u32x4*>(vt + tile_chunk<CH>(key, q) * 8) = in ? cur.v[i] : u32x4{0, 0, 0, 0};
                }
                __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
                __builtin_amdgcn_wave_barrier();
                __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
                for (int c = 0; c < VC; c++) {
                    const float4_t sum = pv(c, float4_t{0.f, 0.f, 0.f, 0.f});
                    if (row == r) o[c] += sum;
                }
                __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
                __builtin_amdgcn_wave_barrier();
                __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        if (pg + W < pg_end) cur = nxt;
    }
    lsum = rows4_sum(lsum);
    __syncthreads();  // the tiles' LDS becomes `red`
    if (has) {
        if (rg == 0) *reinterpret_cast<float2*>(&red[wave][col][0]) = float2{m, lsum * kPUnscale};
#pragma unroll
        for (int c = 0; c < VC; c++)
            *reinterpret_cast<float4_t*>(&red[wave][col][4 + c * 16 + 4 * rg]) = o[c] * (kPUnscale * vref);
    }
    __syncthreads();
#pragma unroll
    for (int g = 0; g < PG; g++) {
        const uint32_t t = threadIdx.x + 64 * W * g, sl = t / (D / 4), d = t % (D / 4) * 4;
        if (sl >= it.ns) continue;
        float M = pm[g];
#pragma unroll
        for (int w = 0; w < W; w++) M = fmaxf(M, red[w][sl][0]);
        const float pw = fast_exp2(pm[g] - M);
        float L = pl[g] * pw;
        float4_t O = po[g] * pw;
#pragma unroll
        for (int w = 0; w < W; w++) {
            const float wt = fast_exp2(red[w][sl][0] - M);
            L += red[w][sl][1] * wt;
            O += *reinterpret_cast<const float4_t*>(&red[w][sl][4 + d]) * wt;
        }
        if (it.part0 == kNoSlot) {
            const uint32_t r = (it.slot0 + sl) / a.group, gg = it.slot0 + sl - r * a.group;
            *reinterpret_cast<float4_t*>(a.out + (int64_t)lay * a.out_layer_stride +
                                         (int64_t)(it.row0 + r) * a.out_row_stride + (head * a.group + gg) * D + d) = O / L;
        } else {
            const uint64_t part = ((uint64_t)(it.part0 + sl) * a.n_lay + lay) * H + head;
            *reinterpret_cast<float4_t*>(a.part_o + part * D + d) = O;
            if (d == 0) *reinterpret_cast<float2*>(a.part_ml + 2 * part) = float2{M, L};
        }
    }
}

// Items of one row's own keys and up to NS slots (a row's query heads of one
// cache head), on the vector units: fewer instructions a page than tiles of 16
// slots that stay nearly empty.  A lane holds 16 bytes of a key row (8 dims, of the
// Q8 cache 16; LPK lanes a row, KPL rows a load), a group of lanes its own softmax
// state over the rows it sees; q.k and p.v mix f32 with the cache's f16 or int8.
// Groups and waves start from the prefix's partials, every (W KPL)-th a group, and
// are joined at the end.
// Bound by memory: 12 layers x 64 rows of 1..255 keys x 12 heads x 64, 316 MB of
// f16 in 55 us (5.8 TB/s).
template <int D, int NS, int W, int INL, bool Q8>
__global__ __launch_bounds__(64 * W) void prefix_rows_kernel(const PrefixLaunch a, const PlanArg<INL> pa) {
    constexpr int DL = Q8 ? 16 : 8;          // dims of a lane
    constexpr int LPK = D / DL;              // lanes of a key row
    constexpr int KPL = 64 / LPK;            // rows of a load
    constexpr int LPP = (int)kPage / KPL;    // loads of a page
    constexpr int PB = D == 64 ? 2 : 1;      // pages of an iteration
    __shared__ float red[W][NS][D + 2];
    const int lane = threadIdx.x & 63;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t H = a.pool.n_head, lh = a.n_lay * H;
    const uint8_t* plan = plan_base(pa, a.plan);
    const uint32_t item_i = blockIdx.x / lh;
    const uint32_t rem = blockIdx.x - item_i * lh;
    const uint32_t lay = rem / H, head = rem - lay * H;
    const PrefixItem it = reinterpret_cast<const PrefixItem*>(plan + a.off_items)[item_i];
    const int kl = lane / LPK, ds = lane % LPK;
    const uint64_t off = (uint64_t)(a.layer0 + lay) * a.pool.layer_halves + (uint64_t)head * a.pool.head_halves;
    const uint32_t* __restrict__ tab = reinterpret_cast<const uint32_t*>(plan + a.off_table) + it.tab;
    const uint32_t pg_end = (it.kv_end + kPage - 1) / kPage;
    struct Regs {
        u32x4 k[PB][LPP], v[PB][LPP];
        float ks[Q8 ? PB : 1][LPP], vs[Q8 ? PB : 1][LPP];  // Q8: the rows' scales
    };
    auto load = [&](uint32_t pg, Regs& r) {
#pragma unroll
        for (int b = 0; b < PB; b++) {
            // (a page past the end: the last again, its keys masked)
            const uint64_t at = off + (uint64_t)tab[min(pg + b, pg_end - 1)] * a.pool.page_halves;
            const u32x4* kp = reinterpret_cast<const u32x4*>(a.pool.k + at) + lane;
            const u32x4* vp = reinterpret_cast<const u32x4*>(a.pool.v + at) + lane;
#pragma unroll
            for (int i = 0; i < LPP; i++) r.k[b][i] = load16(kp + 64 * i);
#pragma unroll
            for (int i = 0; i < LPP; i++) r.v[b][i] = load16(vp + 64 * i);
            if constexpr (Q8) {
#pragma unroll
                for (int i = 0; i < LPP; i++) {
                    r.ks[b][i] = reinterpret_cast<const float*>(q8_block(a.pool, false, at) + kPage * D)[i * KPL + kl];
                    r.vs[b][i] = reinterpret_cast<const float*>(q8_block(a.pool, true, at) + kPage * D)[i * KPL + kl];
                }
            }
        }
    };
    auto value = [](const u32x4& x, int e) {  // dim e of a lane's 16 bytes
        if constexpr (Q8)
            return i8f(x[e / 4], e % 4);
        else
            return (float)__builtin_bit_cast(half8_t, x)[e];
    };
    Regs cur;
    uint32_t pg = it.kv_begin / kPage + wave * PB;
    if (pg < pg_end) load(pg, cur);
    float q[NS][DL], m[NS], l[NS], o[NS][DL];
    {
        // slot s of a row is query head s of the cache head (past ns: the first again, its result unused)
        const float* qb = a.q + (int64_t)lay * a.q_layer_stride + (int64_t)it.row0 * a.q_row_stride +
                          (head * a.group + it.slot0) * D + ds * DL;
#pragma unroll
        for (int s = 0; s < NS; s++) {
            const float* p = qb + (s < (int)it.ns ? s : 0) * D;
#pragma unroll
            for (int e = 0; e < DL; e += 4) {
                const float4 x = *reinterpret_cast<const float4*>(p + e);
                q[s][e] = x.x * a.qscale;
                q[s][e + 1] = x.y * a.qscale;
                q[s][e + 2] = x.z * a.qscale;
                q[s][e + 3] = x.w * a.qscale;
            }
            m[s] = kMinScore;
            l[s] = 0.f;
#pragma unroll
            for (int e = 0; e < DL; e++) o[s][e] = 0.f;
        }
    }
    if (it.part0 == kNoSlot) {
        for (uint32_t j = wave * KPL + kl; j < it.n_pre; j += W * KPL) {
#pragma unroll
            for (int s = 0; s < NS; s++) {
                const uint32_t idx = it.pre0 + (s < (int)it.ns ? s : 0) + j * it.pre_stride;
                const uint64_t part = ((uint64_t)idx * a.n_lay + lay) * H + head;
                const float2 ml = *reinterpret_cast<const float2*>(a.part_ml + 2 * part);
                float4 x[DL / 4];
#pragma unroll
                for (int e = 0; e < DL / 4; e++) x[e] = reinterpret_cast<const float4*>(a.part_o + part * D + ds * DL)[e];
                const float mn = fmaxf(m[s], ml.x);
                const float keep = fast_exp2(m[s] - mn), take = fast_exp2(ml.x - mn);
                m[s] = mn;
                l[s] = l[s] * keep + ml.y * take;
#pragma unroll
                for (int e = 0; e < DL / 4; e++) {
                    o[s][4 * e] = o[s][4 * e] * keep + x[e].x * take;
                    o[s][4 * e + 1] = o[s][4 * e + 1] * keep + x[e].y * take;
                    o[s][4 * e + 2] = o[s][4 * e + 2] * keep + x[e].z * take;
                    o[s][4 * e + 3] = o[s][4 * e + 3] * keep + x[e].w * take;
                }
            }
        }
    }
    for (; pg < pg_end; pg += W * PB) {
        Regs nxt;
        if (pg + W * PB < pg_end) load(pg + W * PB, nxt);
        if ((pg + PB) * kPage > it.kv_end) {
            // Rows past the end: their scores are -inf below, and whatever V
            // holds there may not meet a weight, not even 0.
#pragma unroll
            for (int b = 0; b < PB; b++)
#pragma unroll
                for (int i = 0; i < LPP; i++)
                    if ((pg + b) * kPage + i * KPL + kl >= it.kv_end) {
                        if constexpr (Q8)
                            cur.vs[b][i] = 0.f;
                        else
                            cur.v[b][i] = u32x4{0, 0, 0, 0};
                    }
        }
#pragma unroll
        for (int s = 0; s < NS; s++) {
            float sc[PB][LPP], mx = m[s];
#pragma unroll
            for (int b = 0; b < PB; b++)
#pragma unroll
                for (int i = 0; i < LPP; i++) {
                    float x = 0.f, y = 0.f;
#pragma unroll
                    for (int e = 0; e < DL; e += 2) {
                        x += q[s][e] * value(cur.k[b][i], e);
                        y += q[s][e + 1] * value(cur.k[b][i], e + 1);
                    }
                    x = key_sum<LPK>(x + y);
                    if constexpr (Q8) x *= cur.ks[b][i];
                    sc[b][i] = (pg + b) * kPage + i * KPL + kl < it.kv_end ? x : -INFINITY;
                    mx = fmaxf(mx, sc[b][i]);
                }
            const float keep = fast_exp2(m[s] - mx);
            m[s] = mx;
            l[s] *= keep;
#pragma unroll
            for (int e = 0; e < DL; e++) o[s][e] *= keep;
#pragma unroll
            for (int b = 0; b < PB; b++)
#pragma unroll
                for (int i = 0; i < LPP; i++) {
                    float p = fast_exp2(sc[b][i] - mx);
                    l[s] += p;
                    if constexpr (Q8) p *= cur.vs[b][i];
#pragma unroll
                    for (int e = 0; e < DL; e++) o[s][e] += p * value(cur.v[b][i], e);
                }
        }
        if (pg + W * PB < pg_end) cur = nxt;
    }
    // The wave's groups, then the waves.
#pragma unroll
    for (int s = 0; s < NS; s++) {
#pragma unroll
        for (int st = LPK; st < 64; st <<= 1) {
            const float m2 = __shfl_xor(m[s], st), l2 = __shfl_xor(l[s], st);
            const float mn = fmaxf(m[s], m2);
            const float a1 = fast_exp2(m[s] - mn), a2 = fast_exp2(m2 - mn);
            m[s] = mn;
            l[s] = l[s] * a1 + l2 * a2;
#pragma unroll
            for (int e = 0; e < DL; e++) o[s][e] = o[s][e] * a1 + __shfl_xor(o[s][e], st) * a2;
        }
        if (kl == 0) {
            if (ds == 0) {
                red[wave][s][0] = m[s];
                red[wave][s][1] = l[s];
            }
#pragma unroll
            for (int e = 0; e < DL; e++) red[wave][s][2 + ds * DL + e] = o[s][e];
        }
    }
    __syncthreads();
    for (uint32_t t = threadIdx.x; t < it.ns * D; t += 64 * W) {
        const uint32_t s = t / D, d = t - s * D;
        float M = red[0][s][0];
#pragma unroll
        for (int w = 1; w < W; w++) M = fmaxf(M, red[w][s][0]);
        float L = 0.f, O = 0.f;
#pragma unroll
        for (int w = 0; w < W; w++) {
            const float wt = fast_exp2(red[w][s][0] - M);
            L += red[w][s][1] * wt;
            O += red[w][s][2 + d] * wt;
        }
        if (it.part0 == kNoSlot) {
            a.out[(int64_t)lay * a.out_layer_stride + (int64_t)it.row0 * a.out_row_stride +
                  (head * a.group + it.slot0 + s) * D + d] = O / L;
        } else {
            const uint64_t part = ((uint64_t)(it.part0 + s) * a.n_lay + lay) * H + head;
            a.part_o[part * D + d] = O;
            if (d == 0) {
                a.part_ml[2 * part] = M;
                a.part_ml[2 * part + 1] = L;
            }
        }
    }
}

// Wide items: W waves of 32 slots each, KG times over, over tiles of 32 keys of a
// prefix.  Each group of W waves takes every KG-th tile: it copies them to LDS by
// DMA (a ring of four tiles, one barrier a tile), and all its waves read them.  The
// groups' states are joined at the end.  Of the 32 x 32 x 16 products S^T = K Q^T and O^T += V^T P^T lane l
// holds slot l % 32: a slot's softmax state lives in two lanes, and S^T's
// registers are PV's operand as they are (keys 8 (i / 4) + 4 (l / 32) + i % 4 of
// register i, in V's transposing reads alike).  Every slot sees every key, so
// only the last tile masks.  The exponent reference follows the running maximum
// only past kWideSlack (weights up to 2^15 in f16, as hi + lo).
// 192 slots x 8 heads x 128 behind 8185 keys (three waves, two groups): 26.5 us, of
// which ~5 until the first tile is there, ~3 to join and store, ~4 until the
// partials have left the caches, and between them ~2 us per two tiles, half of it
// matrix products on the SIMDs that hold two of the six waves.
constexpr float kWideSlack = 8.f, kWideLog2 = 7.f, kWideUnscale = 1.f / 128.f;
typedef float float16_t __attribute__((ext_vector_type(16)));
typedef int v2i32_t __attribute__((ext_vector_type(2)));

// 4 bytes per lane from g to LDS at lds + 4 * lane (as lds_dma16).
__device__ __forceinline__ void lds_dma4(uint64_t g, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dword %0, off" : : "v"(g), "s"(lds) : "memory", "m0");
}

template <int N>
__device__ __forceinline__ void wait_dma(uint32_t ahead) {  // at most `ahead` tiles of N copies of this wave in flight
    static_assert(N < 64, "vmcnt");
    if (ahead >= 1)
        __builtin_amdgcn_s_waitcnt(0x0f70 | (N & 15) | ((N >> 4) << 14));
    else
        __builtin_amdgcn_s_waitcnt(0x0f70);
}

//
// Q8: the int8 rows are copied as they are, their 64 scales beside them, and
// become f16 on their way to the products; key scales multiply the scores, value
// scales the weights (in units of vref, as in prefix_attn_kernel).
template <int D, int W, int KG, bool Q8, int INL>
__global__ __launch_bounds__(64 * W * KG) __attribute__((amdgpu_waves_per_eu(D == 128 ? 2 : 3, 8)))
void prefix_wide_kernel(const PrefixLaunch a, const PlanArg<INL> pa) {
    constexpr int KS = D / 16;                // 16-dim steps of QK
    constexpr int DB = D / 32;                // 32-dim blocks of PV
    constexpr int RB = Q8 ? D : 2 * D;        // bytes of a row
    constexpr int CH = RB / 16;               // 16-byte chunks of a row
    constexpr int TP = 2, TK = TP * kPage;    // pages and keys of a tile
    constexpr int TB = TK * RB;               // bytes of a K (or V) tile
    constexpr int SB = 2 * TB + (Q8 ? 256 : 0);  // of a stage: K, V, and scales [page][K|V][16]
    constexpr int NI = 2 * TB / 1024;         // 1 KB copies of a tile
    constexpr int ND = (NI + W - 1) / W;      // of one wave (the last again, where they do not divide)
    constexpr int NW = ND + (Q8 ? 1 : 0);     // loads of one wave: the scales by every wave
    constexpr int WR = 64 / CH;               // rows of one copy
    constexpr int NS = 4;                     // tiles of the ring
    constexpr float kHi = kWideSlack + kWideLog2;
    constexpr size_t kStates = (size_t)(KG - 1) * W * (16 * DB + 3) * 64 * 4;
    constexpr size_t kRing = (size_t)KG * NS * SB > kStates ? (size_t)KG * NS * SB : kStates;
    constexpr int SW = 16 * DB + 3;           // a lane's state: o, then its slot's m, l and vref
    __shared__ __attribute__((aligned(16))) uint8_t lds[kRing];

    const int lane = threadIdx.x & 63;
    const uint32_t wave_all = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t kg = wave_all / W, wave = wave_all - kg * W;  // group of keys, wave of slots
    uint8_t(*const ring)[SB] = reinterpret_cast<uint8_t(*)[SB]>(lds + kg * NS * SB);
    const uint32_t H = a.pool.n_head, lh = a.n_lay * H;
    const uint8_t* plan = plan_base(pa, a.plan);
    const uint32_t item_i = blockIdx.x / lh;
    const uint32_t rem = blockIdx.x - item_i * lh;
    const uint32_t lay = rem / H, head = rem - lay * H;
    const PrefixItem it = reinterpret_cast<const PrefixItem*>(plan + a.off_items)[item_i];
    const int col = lane & 31, g2 = lane >> 5;
    const uint64_t off = (uint64_t)(a.layer0 + lay) * a.pool.layer_halves + (uint64_t)head * a.pool.head_halves;
    const uint8_t* kbase = reinterpret_cast<const uint8_t*>(a.pool.k + off);
    const uint8_t* vbase = reinterpret_cast<const uint8_t*>(a.pool.v + off);
    const uint64_t page_bytes = 2 * a.pool.page_halves;
    const __attribute__((address_space(4))) uint32_t* tab =
        (const __attribute__((address_space(4))) uint32_t*)(plan + a.off_table) + it.tab;
    // The group's tiles: every KG-th of the item's.
    const uint32_t pg0 = it.kv_begin / kPage + kg * TP, pg_end = (it.kv_end + kPage - 1) / kPage;
    const uint32_t all_tiles = (pg_end - it.kv_begin / kPage + TP - 1) / TP;
    const uint32_t n_tiles = (all_tiles + KG - 1 - kg) / KG;
    constexpr uint32_t PS = KG * TP;  // pages from a tile of the group to its next

    // Copy i of a tile: rows (i % (NI/2)) * WR .. of K (i < NI/2) or V.  Lane
    // l's 16 bytes land at 16 l of the copy's 1 KB: logical chunk (l % CH) ^ sw
    // of row l / CH.  A row past the item's end copies row 0 of its page, a
    // page past it the item's last page: keys of the item, whose weights the
    // last tile makes 0.
    // (A copy's row and swizzle are bits of their own above the lane's, so its
    // offsets are the lane's in copy 0 with the copy's bits flipped.)
    auto swizzle = [](uint32_t row) -> uint32_t {  // chunk q of a row lies at q ^ swizzle(row)
        if constexpr (Q8)
            return D == 64 ? (row >> 2) & 3 : (row >> 1) & 7;  // the 32 rows of a K operand, 16 of V's: distinct banks
        else
            return tile_chunk<CH>(row, 0) - row * CH;
    };
    const uint32_t lds_ring = (uint32_t)(uintptr_t)NI_LDS(&ring[0][0]);
    const uint32_t lane_o = (uint32_t)(lane / CH) * RB + ((lane % CH) ^ swizzle(lane / CH)) * 16;
    // Q8: lane's scale of page lane / 32, K or V (lane / 16 % 2), position lane % 16.
    const uint64_t scale_from = reinterpret_cast<uint64_t>(lane & 16 ? vbase : kbase) + kPage * D + 4 * (lane & 15);
    uint32_t flip[ND], row0[ND], to[ND];  // of this wave's copies (kept in scalars: the same in every tile)
    uint64_t from[ND];
#pragma unroll
    for (int j = 0; j < ND; j++) {
        const uint32_t i = min(wave + j * W, (uint32_t)NI - 1);
        row0[j] = (i % (NI / 2)) * WR;
        const uint32_t rp = row0[j] % kPage;
        flip[j] = rp * RB | swizzle(rp) * 16;
        to[j] = lds_ring + 1024 * i;
        from[j] = reinterpret_cast<uint64_t>(i >= NI / 2 ? vbase : kbase);
        asm volatile("" : "+s"(flip[j]), "+s"(row0[j]), "+s"(to[j]), "+s"(from[j]));
    }
    uint32_t pid0 = 0, pid1 = 0;  // the pages of the tile to copy next, asked for a tile ahead
    auto pages = [&](uint32_t ti) {
        if (ti < n_tiles) {
            pid0 = tab[pg0 + ti * PS];
            pid1 = tab[min(pg0 + ti * PS + 1, pg_end - 1)];
        }
    };
    auto issue = [&](uint32_t stage, uint32_t ti) {
        const uint32_t pg = pg0 + ti * PS;
        const uint64_t pb0 = pid0 * page_bytes, pb1 = pid1 * page_bytes;
        pages(ti + 1);
        const bool cut = (pg + TP) * kPage > it.kv_end;
#pragma unroll
        for (int j = 0; j < ND; j++) {
            uint32_t o = lane_o ^ flip[j];
            if (cut) o = pg * kPage + row0[j] + lane / CH >= it.kv_end ? o & (RB - 1) : o;  // row 0 of the page
            lds_dma16_sbase(reinterpret_cast<const void*>(from[j] + (row0[j] >= kPage ? pb1 : pb0)), o,
                            to[j] + stage * SB);
        }
        if constexpr (Q8) lds_dma4(scale_from + (lane & 32 ? pb1 : pb0), lds_ring + stage * SB + 2 * TB);
    };
    const uint32_t s0 = wave * kWideSlots;
    const bool mine = s0 < it.ns;  // the wave has slots
    const bool has = s0 + col < it.ns;
    const uint32_t slot = it.slot0 + (has ? s0 + col : 0u);
    const uint32_t row = slot / a.group, gq = slot - row * a.group;
    float4 xq[2 * KS];
    {
        const float* qb = a.q + (int64_t)lay * a.q_layer_stride + (int64_t)(it.row0 + row) * a.q_row_stride +
                          (head * a.group + gq) * D + 8 * g2;
#pragma unroll
        for (int c = 0; c < KS; c++) {
            xq[2 * c] = reinterpret_cast<const float4*>(qb + c * 16)[0];
            xq[2 * c + 1] = reinterpret_cast<const float4*>(qb + c * 16)[1];
        }
    }
    pages(0);
    for (uint32_t t = 0; t < min(n_tiles, (uint32_t)NS - 1); t++) issue(t, t);
    // The loads (and the first tiles, issued after them) have landed before any
    // further copy: the loop's waits count copies alone.
#pragma unroll
    for (int c = 0; c < 2 * KS; c++) asm volatile("" : : "v"(xq[c].x), "v"(xq[c].y), "v"(xq[c].z), "v"(xq[c].w));
    half8_t qh[KS], ql[KS];
#pragma unroll
    for (int c = 0; c < KS; c++) {
        const float x[8] = {xq[2 * c].x, xq[2 * c].y, xq[2 * c].z, xq[2 * c].w,
                            xq[2 * c + 1].x, xq[2 * c + 1].y, xq[2 * c + 1].z, xq[2 * c + 1].w};
        float y[8];
#pragma unroll
        for (int e = 0; e < 8; e++) {
            y[e] = has ? x[e] * a.qscale : 0.f;
            asm("" : "+v"(y[e]));  // the f32 products, as the split's residual sees them
        }
        split8(y, qh[c], ql[c]);
    }
    float mref = 0.f, lsum = 0.f;
    float vref = Q8 ? kMinScale : 1.f, vinv = 1.f / vref;
    bool set = false;  // the reference is a score's (alike in both lanes of a slot)
    float16_t o[DB];
#pragma unroll
    for (int b = 0; b < DB; b++)
#pragma unroll
        for (int i = 0; i < 16; i++) o[b][i] = 0.f;
    // Byte offsets in a stage: K chunk 2c + g2 of row col; V keys 8j + 4 g2 +
    // (0..3), dims 32 b + 16 (l / 16 % 2) + (0..15) of a page.
    // (Q8: 8 bytes of K's chunk c; V's keys of both j in one 8-bit transposing
    // read, whose lane 2e + a of 16 reads bytes 8a .. of row e and lane j receives
    // byte j of the eight rows.)
    uint32_t koff[KS], voff[Q8 ? 1 : 2][DB];
    const int vt = (lane >> 2) & 3, va = lane & 3, vh = (lane >> 4) & 1;
#pragma unroll
    for (int c = 0; c < KS; c++)
        koff[c] = Q8 ? col * RB + (c ^ swizzle(col)) * 16 + 8 * g2 : col * RB + ((2 * c + g2) ^ swizzle(col)) * 16;
#pragma unroll
    for (int b = 0; b < DB; b++) {
        if constexpr (Q8) {
            const uint32_t e = (lane & 15) >> 1, key = (e < 4 ? 0 : 8) + 4 * g2 + (e & 3);
            voff[0][b] = TB + key * RB + ((2 * b + vh) ^ swizzle(key)) * 16 + 8 * (lane & 1);
        } else {
#pragma unroll
            for (int j = 0; j < 2; j++) {
                const uint32_t key = 8 * j + 4 * g2 + vt;
                voff[j][b] = TB + key * RB + ((4 * b + 2 * vh + (va >> 1)) ^ swizzle(key)) * 16 + (va & 1) * 8;
            }
        }
    }
    auto key_operand = [&](const uint8_t* st, int c) -> half8_t {
        if constexpr (Q8) {
            const uint2 w = *reinterpret_cast<const uint2*>(st + koff[c]);
            return __builtin_shufflevector(i8x4_f16(w.x), i8x4_f16(w.y), 0, 1, 2, 3, 4, 5, 6, 7);
        } else {
            return *reinterpret_cast<const half8_t*>(st + koff[c]);
        }
    };
    // Q8: the scales of the lane's 16 keys, K's (which = 0) or V's.
    auto scales = [&](uint32_t stage, int which, float (&x)[16]) {
        const uint8_t* p = &ring[stage][0] + 2 * TB + 64 * which + 16 * g2;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float4 y = *reinterpret_cast<const float4*>(p + (i / 2) * 128 + (i % 2) * 32);
            x[4 * i] = y.x;
            x[4 * i + 1] = y.y;
            x[4 * i + 2] = y.z;
            x[4 * i + 3] = y.w;
        }
    };

    // S^T of the tile at `stage`, relative to the reference, with `between(c)`
    // written behind the products of step c: work that does not depend on them.
    auto scores = [&](uint32_t stage, auto between) {
        const uint8_t* const st = &ring[stage][0];
        float16_t sc;
#pragma unroll
        for (int i = 0; i < 16; i++) sc[i] = Q8 ? 0.f : -mref;
        half8_t kh[4];
#pragma unroll
        for (int c = 0; c < 4; c++) kh[c] = key_operand(st, c);
#pragma unroll
        for (int c = 0; c < KS; c++) {
            sc = __builtin_amdgcn_mfma_f32_32x32x16_f16(kh[c % 4], ql[c], sc, 0, 0, 0);
            sc = __builtin_amdgcn_mfma_f32_32x32x16_f16(kh[c % 4], qh[c], sc, 0, 0, 0);
            asm volatile("" : "+v"(sc));  // the products stay here, not where their sum is used
            if (c + 4 < KS) kh[c % 4] = key_operand(st, c + 4);
            between(c);
            __builtin_amdgcn_sched_barrier(0);
        }
        if constexpr (Q8) {
            float ks[16];
            scales(stage, 0, ks);
#pragma unroll
            for (int i = 0; i < 16; i++) sc[i] = fmaf(sc[i], ks[i], -mref);
        }
        return sc;
    };
    auto largest = [](const float16_t& sc) {
        float lm = sc[0];
#pragma unroll
        for (int i = 1; i < 16; i++) lm = fmaxf(lm, sc[i]);
        return lm;
    };
    // V's operand for keys of page t of the tile at `st`.
    auto values = [&](const uint8_t* st, int t, half8_t (&v8)[DB]) {
#pragma unroll
        for (int b = 0; b < DB; b++) {
            if constexpr (Q8) {
                const v2i32_t r = __builtin_amdgcn_ds_read_tr8_b64_v2i32(
                    (__attribute__((address_space(3))) v2i32_t*)(st + voff[0][b] + t * (int)kPage * RB));
                const half4_t lo = i8x4_f16((uint32_t)r.x), hi = i8x4_f16((uint32_t)r.y);
                v8[b] = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
            } else {
                half4_t v[2];
#pragma unroll
                for (int j = 0; j < 2; j++)
                    v[j] = __builtin_bit_cast(
                        half4_t, __builtin_amdgcn_ds_read_tr16_b64_v4f16((__attribute__((address_space(3))) v4fp16_t*)(
                                     st + voff[j][b] + t * (int)kPage * RB)));
                v8[b] = __builtin_shufflevector(v[0], v[1], 0, 1, 2, 3, 4, 5, 6, 7);
            }
        }
    };
    float16_t sc;
    float lm = 0.f;  // the lane's largest score
    // Tile ti: its weights are taken while the products of tile ti + 1's scores
    // run, so that neither the vector nor the matrix units wait for the other.
    auto tile = [&](auto lastc, uint32_t stage, uint32_t ti) {
        constexpr bool LAST = decltype(lastc)::value;
        const uint8_t* const st = &ring[stage][0];
        if constexpr (LAST) {
            const uint32_t key0 = (pg0 + ti * PS) * kPage;
            if (key0 + TK > it.kv_end) {
#pragma unroll
                for (int i = 0; i < 16; i++)
                    if (key0 + 8 * (i / 4) + 4 * g2 + i % 4 >= it.kv_end) sc[i] = -INFINITY;
            }
        }
        if constexpr (LAST) lm = largest(sc);
        if (__any(lm > kHi || !set)) {
            const u32x2_t sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(lm), __float_as_uint(lm), false, false);
            const float mx = fmaxf(__uint_as_float(sw[0]), __uint_as_float(sw[1])) - kWideLog2;
            // The first finite maximum sets the reference, later ones only raise it.
            const bool none = mx == -INFINITY;
            const float d = set ? fmaxf(mx, 0.f) : none ? 0.f : mx;
            const float alpha = set ? fast_exp2(-d) : 1.f;  // (nothing is summed yet)
            set = set || !none;
            lsum *= alpha;
#pragma unroll
            for (int b = 0; b < DB; b++) o[b] *= alpha;
            mref += d;
#pragma unroll
            for (int i = 0; i < 16; i++) sc[i] -= d;
        }
        float vs[Q8 ? 16 : 1];
        if constexpr (Q8) {
            scales(stage, 1, vs);
            if constexpr (LAST) {  // scales past the end may be anything
                const uint32_t key0 = (pg0 + ti * PS) * kPage;
#pragma unroll
                for (int i = 0; i < 16; i++)
                    if (key0 + 8 * (i / 4) + 4 * g2 + i % 4 >= it.kv_end) vs[i] = 0.f;
            }
            float vm = vs[0];
#pragma unroll
            for (int i = 1; i < 16; i++) vm = fmaxf(vm, vs[i]);
            if (__any(vm > vref)) {  // (a scale belongs to its key: the same for every slot)
                const uint32_t bits = __float_as_uint(vm);
                const u32x2_t sw = __builtin_amdgcn_permlane32_swap(bits, bits, false, false);
                vm = fmaxf(scale_reference(fmaxf(__uint_as_float(sw[0]), __uint_as_float(sw[1]))), vref);
                const float shrink = vref / vm;
                vref = vm;
                vinv = 1.f / vm;
#pragma unroll
                for (int b = 0; b < DB; b++) o[b] *= shrink;
            }
        }
        float ps[4] = {0.f, 0.f, 0.f, 0.f};
        u32x4 ph[TP], pl[TP];
        auto weights = [&](int c) {  // values 16 c / KS .. of the 16, in pairs
            constexpr int N = 16 / KS;
#pragma unroll
            for (int i = c * N; i < (c + 1) * N; i += 2) {
                float p0 = fast_exp2(sc[i]), p1 = fast_exp2(sc[i + 1]);
                ps[(i / 2) % 4] += p0 + p1;
                if constexpr (Q8) {
                    p0 *= vs[i] * vinv;
                    p1 *= vs[i + 1] * vinv;
                }
                uint32_t h, l;
                split_w16x2(p0, p1, h, l);
                ph[i / 8][i % 8 / 2] = h;
                pl[i / 8][i % 8 / 2] = l;
            }
        };
        float16_t next;
        half8_t v8[TP][DB];
        values(st, 0, v8[0]);
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (LAST) {
#pragma unroll
            for (int c = 0; c < KS; c++) weights(c);
        } else {
            next = scores((stage + 1) % NS, weights);
        }
        lsum += (ps[0] + ps[1]) + (ps[2] + ps[3]);
        settle(ph[0], pl[0], ph[1], pl[1]);
        values(st, 1, v8[1]);
#pragma unroll
        for (int t = 0; t < TP; t++) {
            const half8_t p_hi = __builtin_bit_cast(half8_t, ph[t]), p_lo = __builtin_bit_cast(half8_t, pl[t]);
#pragma unroll
            for (int b = 0; b < DB; b++) o[b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v8[t][b], p_lo, o[b], 0, 0, 0);
#pragma unroll
            for (int b = 0; b < DB; b++) o[b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v8[t][b], p_hi, o[b], 0, 0, 0);
        }
        static_assert(TP == 2, "two pages of V operands");
        if constexpr (!LAST) {
            sc = next;
            lm = largest(sc);
        }
    };
    const bool busy = mine && n_tiles > 0;
    wait_dma<NW>(0);
    __syncthreads();  // tile 0 is there
    if (busy) {
        sc = scores(0, [](int) {});
        lm = largest(sc);
    }
    // (the stage is a variable: the body instantiated per stage spills many
    // registers at head_dim 128, where three waves of f16 spill 12 bytes a lane as it
    // is, and two of Q8 8)
    uint32_t stage = 0;
    const uint32_t steps = (all_tiles + KG - 1) / KG;
    for (uint32_t ti = 0; ti + 1 < steps; ti++) {
        wait_dma<NW>(ti + 2 < n_tiles ? 1 : 0);
        __syncthreads();  // every wave's part of tile ti + 1 is there, and every wave is done with tile ti - 1
        if (ti + NS - 1 < n_tiles) issue((ti + NS - 1) % NS, ti + NS - 1);
        if (busy && ti + 1 < n_tiles) {
            tile(std::false_type{}, stage, ti);
            stage = (stage + 1) % NS;
        }
    }
    // (a group with a tile less has kept its last one for here)
    if (busy) tile(std::true_type{}, stage, n_tiles - 1);
    const u32x2_t sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(lsum), __float_as_uint(lsum), false, false);
    lsum = __uint_as_float(sw[0]) + __uint_as_float(sw[1]);
    if constexpr (KG > 1) {  // the other groups' states through LDS to the first
        __syncthreads();  // every group is done with the ring
        float* const box = reinterpret_cast<float*>(lds) + wave * SW * 64 + lane;
        constexpr int GS = W * SW * 64;  // floats of a group
        if (kg > 0) {
            float* p = box + (kg - 1) * GS;
#pragma unroll
            for (int b = 0; b < DB; b++)
#pragma unroll
                for (int i = 0; i < 16; i++) p[(16 * b + i) * 64] = o[b][i];
            p[16 * DB * 64] = set ? mref : kMinScore;
            p[(16 * DB + 1) * 64] = lsum;
            p[(16 * DB + 2) * 64] = vref;
        }
        __syncthreads();
        if (kg > 0) return;
#pragma unroll
        for (int g = 0; g < KG - 1; g++) {
            const float* p = box + g * GS;
            const float m2 = p[16 * DB * 64];
            const float m1 = set ? mref : kMinScore, mn = fmaxf(m1, m2);
            const float w1 = fast_exp2(m1 - mn), w2 = fast_exp2(m2 - mn);
            if (mn > kMinScore) {
                mref = mn;
                set = true;
            }
            lsum = lsum * w1 + p[(16 * DB + 1) * 64] * w2;
            float u1 = w1, u2 = w2;
            if constexpr (Q8) {  // in units of the larger vref
                const float v1 = vref, v2 = p[(16 * DB + 2) * 64];
                vref = fmaxf(v1, v2);
                u1 *= v1 / vref;
                u2 *= v2 / vref;
            }
#pragma unroll
            for (int b = 0; b < DB; b++)
#pragma unroll
                for (int i = 0; i < 16; i++) o[b][i] = o[b][i] * u1 + p[(16 * b + i) * 64] * u2;
        }
    }
    if (!has) return;
    const uint64_t part = ((uint64_t)(it.part0 + s0 + col) * a.n_lay + lay) * H + head;
    if (g2 == 0) {
        a.part_ml[2 * part] = set ? mref + kWideLog2 : kMinScore;
        a.part_ml[2 * part + 1] = lsum * kWideUnscale;
    }
#pragma unroll
    for (int b = 0; b < DB; b++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
            float4 y;
            const float unit = kWideUnscale * vref;
            y.x = o[b][4 * i] * unit;
            y.y = o[b][4 * i + 1] * unit;
            y.z = o[b][4 * i + 2] * unit;
            y.w = o[b][4 * i + 3] * unit;
            *reinterpret_cast<float4*>(a.part_o + part * D + 32 * b + 8 * i + 4 * g2) = y;
        }
}

// One wave per (row, layer, query head): its partials' states weighed by
// exp2(m - M) and added; lane l holds dims l, l + 64.  4-5 us, the plan's item, the
// states and the sums one after another, with little to read.
template <int D, int INL>
__global__ __launch_bounds__(64 * kMergeWaves) void prefix_merge_kernel(const PrefixLaunch a, const PlanArg<INL> pa) {
    constexpr int N = D / 64;
    const uint32_t lane = threadIdx.x & 63u;
    const uint32_t H = a.pool.n_head, hq = H * a.group;
    const uint64_t unit = (uint64_t)blockIdx.x * kMergeWaves + (threadIdx.x >> 6);
    const uint64_t per = (uint64_t)a.n_lay * hq;
    if (unit >= per * a.n_merges) return;
    const uint32_t mi = (uint32_t)(unit / per);
    const uint32_t rem = (uint32_t)(unit - (uint64_t)mi * per);
    const uint32_t lay = rem / hq, qhead = rem - lay * hq;
    const uint32_t head = qhead / a.group, g = qhead - head * a.group;
    const PrefixMerge me = reinterpret_cast<const PrefixMerge*>(plan_base(pa, a.plan) + a.off_merges)[mi];
    auto part_of = [&](uint32_t i) {
        const uint32_t idx = i < me.n_own ? me.own0 + i * me.own_stride : me.pre0 + (i - me.n_own) * me.pre_stride;
        return ((uint64_t)(idx + g) * a.n_lay + lay) * H + head;
    };
    const uint32_t n = me.n_own + me.n_pre;
    float M = kMinScore, L = 0.f, O[N] = {};
    for (uint32_t i0 = 0; i0 < n; i0 += 64) {  // 64 partials' (m, l) at a time, one a lane
        const uint32_t cnt = min(64u, n - i0);
        float m = kMinScore, l = 0.f;
        if (lane < cnt) {
            const float2 ml = *reinterpret_cast<const float2*>(a.part_ml + 2 * part_of(i0 + lane));
            m = ml.x;
            l = ml.y;
        }
        float mx = m;
        for (int off = 32; off > 0; off >>= 1) mx = fmaxf(mx, __shfl_xor(mx, off));
        const float mn = fmaxf(M, mx);
        const float alpha = fast_exp2(M - mn);
        M = mn;
        const float w = fast_exp2(m - mn);
        float ls = l * w;
        for (int off = 32; off > 0; off >>= 1) ls += __shfl_xor(ls, off);
        L = L * alpha + ls;
#pragma unroll
        for (int e = 0; e < N; e++) O[e] *= alpha;
        constexpr int B = 8;  // partials in flight; past the last it is read again and weighs nothing
        for (uint32_t i = 0; i < cnt; i += B) {
            float x[B][N];
#pragma unroll
            for (int j = 0; j < B; j++) {
                const float* p = a.part_o + part_of(i0 + min(i + j, cnt - 1)) * D + lane;
#pragma unroll
                for (int e = 0; e < N; e++) x[j][e] = p[64 * e];
            }
#pragma unroll
            for (int j = 0; j < B; j++) {
                const float wi = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(w), (int)min(i + j, 63u)));
#pragma unroll
                for (int e = 0; e < N; e++)
                    if (i + j < cnt) O[e] += x[j][e] * wi;
            }
        }
    }
    float* dst = a.out + (int64_t)lay * a.out_layer_stride + (int64_t)me.row * a.out_row_stride + qhead * D + lane;
#pragma unroll
    for (int e = 0; e < N; e++) dst[64 * e] = O[e] / L;
}

// One workgroup per (item, layer, head): prefix_attn_kernel or prefix_rows_kernel.
template <int D>
hipError_t items_t(const PrefixLaunch& a, const void* ip, uint32_t ib, hipStream_t s, const LaunchTiming& t) {
    const uint64_t blocks = (uint64_t)a.n_items * a.n_lay * a.pool.n_head;
    return with_plan(a, ip, ib, [&](auto pa) {
        constexpr int INL = sizeof(pa.b) > 4 ? (int)sizeof(pa.b) : 0;
        auto run = [&](auto q8) {
            constexpr bool Q8 = decltype(q8)::value;
            if (a.row_slots == 1) {
                if (a.waves == 2) return go(prefix_rows_kernel<D, 1, 2, INL, Q8>, blocks, 128, s, t, a, pa);
                if (a.waves == 4) return go(prefix_rows_kernel<D, 1, 4, INL, Q8>, blocks, 256, s, t, a, pa);
            }
            if constexpr (!Q8) {
                if (a.row_slots == 2 && a.waves == 2) return go(prefix_rows_kernel<D, 2, 2, INL, Q8>, blocks, 128, s, t, a, pa);
                if (a.row_slots == 2 && a.waves == 4) return go(prefix_rows_kernel<D, 2, 4, INL, Q8>, blocks, 256, s, t, a, pa);
            }
            if (a.row_slots) return hipErrorInvalidValue;
            return go(prefix_attn_kernel<D, INL, Q8>, blocks, 64 * kItemWaves, s, t, a, pa);
        };
        return a.pool.q8 ? run(std::true_type{}) : run(std::false_type{});
    });
}

template <int D, bool Q8>
hipError_t wide_t(const PrefixLaunch& a, const void* ip, uint32_t ib, hipStream_t s, const LaunchTiming& t) {
    const uint64_t blocks = (uint64_t)a.n_items * a.n_lay * a.pool.n_head;
    constexpr int K1 = wide_groups(D, 1), K2 = wide_groups(D, 2), K3 = wide_groups(D, 3), K4 = wide_groups(D, 4);
    return with_plan(a, ip, ib, [&](auto pa) {
        constexpr int INL = sizeof(pa.b) > 4 ? (int)sizeof(pa.b) : 0;
        switch (a.waves) {
            case 1: return go(prefix_wide_kernel<D, 1, K1, Q8, INL>, blocks, 64 * K1, s, t, a, pa);
            case 2: return go(prefix_wide_kernel<D, 2, K2, Q8, INL>, blocks, 128 * K2, s, t, a, pa);
            case 3: return go(prefix_wide_kernel<D, 3, K3, Q8, INL>, blocks, 192 * K3, s, t, a, pa);
            case 4: return go(prefix_wide_kernel<D, 4, K4, Q8, INL>, blocks, 256 * K4, s, t, a, pa);
            default: return hipErrorInvalidValue;
        }
    });
}

}  // namespace

hipError_t launch_prefix_attention(const PrefixLaunch& a, const void* ip, uint32_t ib, hipStream_t s,
                                   const LaunchTiming& t) {
    if (a.n_items == 0) return hipSuccess;
    if (a.pool.head_dim != 64 && a.pool.head_dim != 128) return hipErrorInvalidValue;
    if (!a.wide) return a.pool.head_dim == 64 ? items_t<64>(a, ip, ib, s, t) : items_t<128>(a, ip, ib, s, t);
    if (a.pool.head_dim == 64)
        return a.pool.q8 ? wide_t<64, true>(a, ip, ib, s, t) : wide_t<64, false>(a, ip, ib, s, t);
    return a.pool.q8 ? wide_t<128, true>(a, ip, ib, s, t) : wide_t<128, false>(a, ip, ib, s, t);
}

hipError_t launch_prefix_merge(const PrefixLaunch& a, const void* ip, uint32_t ib, hipStream_t s,
                               const LaunchTiming& t) {
    const uint64_t units = (uint64_t)a.n_merges * a.n_lay * a.pool.n_head * a.group;
    if (units == 0) return hipSuccess;
    return with_plan(a, ip, ib, [&](auto pa) {
        constexpr int INL = sizeof(pa.b) > 4 ? (int)sizeof(pa.b) : 0;
        const uint64_t blocks = (units + kMergeWaves - 1) / kMergeWaves;
        if (a.pool.head_dim == 64) return go(prefix_merge_kernel<64, INL>, blocks, 64 * kMergeWaves, s, t, a, pa);
        return go(prefix_merge_kernel<128, INL>, blocks, 64 * kMergeWaves, s, t, a, pa);
    });
}

}  // namespace ni
