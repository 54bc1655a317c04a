// page_kernels.hip -- gfx950 kernel of page copies (ni_kv_fork, ni_kv_reorder,
// ni_kv_own, ni_kv_compact).
//
// A page is one contiguous run of bytes in each layer, so a whole page is copied
// as it lies, in 16-byte units.  Of a page that a sequence ends in, only the rows
// before the end are: of each (head, K|V) block the units of those rows and their
// scales.
#include "kv_device.h"

namespace ni {
namespace {

constexpr int kCT = 256;        // threads
constexpr int kUnits = 4;       // 16-byte units of a thread, loaded before the first is stored
constexpr uint32_t kTileUnits = kCT * kUnits;

// A page's layout in 16-byte units.
struct PageShape {
    uint32_t page;        // of one layer
    uint32_t block;       // of one (head, K|V) block
    uint32_t values;      // of its values, 16 rows
    uint32_t blocks;      // 2 * heads
};

// Workgroup (copy from `first` on, layer, tile of kTileUnits units).  Bound by memory, each
// byte read and written once past the caches (non-temporal: a copied page is not read
// again soon): 477 pages x 4 layers of 256 KB, 1.0 GB moved, 194 us, 5.15 TB/s (torch's copy of 4
// GB 4.8).  Few copies are bound by the launch: 28 part pages x 12 layers of 48 KB 6.6 us, four
// 4.0.  Four units to a thread: all loads of a tile are in flight at once, and a page of 12
// heads is three tiles.
template <int INL>
__global__ __launch_bounds__(kCT) void page_copy_kernel(const PageCopyLaunch a, const PageShape g, const uint32_t tiles,
                                                        const uint32_t first, const PlanArg<INL> pa) {
    const uint32_t unit = blockIdx.x / tiles, tile = blockIdx.x - unit * tiles;
    const uint32_t i = unit / a.n_layer, layer = unit - i * a.n_layer;
    const PageCopy c = reinterpret_cast<const PageCopy*>(plan_base(pa, a.plan))[first + i];
    uint8_t* const base = reinterpret_cast<uint8_t*>(a.pool.k + (uint64_t)layer * a.pool.layer_halves);
    const u32x4* const src = reinterpret_cast<const u32x4*>(base + (uint64_t)c.src * g.page * 16);
    u32x4* const dst = reinterpret_cast<u32x4*>(base + (uint64_t)c.dst * g.page * 16);
    const bool part = c.rows < kPage;
    // Of a part: units of a block's rows, and those with their scales (block-scaled: of
    // a run of 64 dims of K and of V, four positions of V to a unit; its scales end the page).
    const uint32_t values = part ? a.pool.b8 ? 4 * c.rows + 16 * ((c.rows + 3) / 4) : g.values / kPage * c.rows : 0;
    const uint32_t scales = part && a.pool.q8 ? (c.rows + 3) / 4 : 0;
    const uint32_t per = values + scales, runs = a.pool.b8 ? g.blocks / 2 * (g.block / 64) : g.blocks;
    const uint32_t n = part ? per * runs + (a.pool.b8 ? (a.pool.n_head + 1) / 2 : 0) : g.page;
    u32x4 x[kUnits];
    uint32_t at[kUnits], words[kUnits];  // unit of the page; words of it to copy
#pragma unroll
    for (int j = 0; j < kUnits; j++) {
        const uint32_t u = tile * kTileUnits + j * kCT + threadIdx.x;
        at[j] = u;
        words[j] = u < n ? 4 : 0;
        if (part && u < n) {
            const uint32_t b = u / per, w = u - b * per;
            if (!a.pool.b8) {
                at[j] = b * g.block + (w < values ? w : g.values + w - values);
                if (w >= values) words[j] = min(4u, c.rows - 4 * (w - values));
            } else if (b < runs) {
                const uint32_t nb = g.block / 64, head = b / nb, x16 = w / c.rows;
                at[j] = (2 * head * nb + b % nb) * 64 + (w < 4 * c.rows ? x16 * 16 + w - x16 * c.rows : nb * 64 + w - 4 * c.rows);
            } else {
                at[j] = a.pool.b8 / 16 + u - per * runs;
            }
        }
        if (words[j]) x[j] = __builtin_nontemporal_load(src + at[j]);
    }
#pragma unroll
    for (int j = 0; j < kUnits; j++) {
        if (words[j] == 4) {
            __builtin_nontemporal_store(x[j], dst + at[j]);
        } else if (words[j]) {
            uint32_t* p = reinterpret_cast<uint32_t*>(dst + at[j]);
            for (uint32_t w = 0; w < words[j]; w++) p[w] = x[j][w];
        }
    }
}

}  // namespace

hipError_t launch_page_copy(const PageCopyLaunch& a, const void* ip, uint32_t ib, hipStream_t s) {
    PageShape g;
    g.page = (uint32_t)(a.pool.page_halves / 8);
    g.block = a.pool.head_halves / 16;
    g.values = kPage * a.pool.head_dim / (a.pool.q8 ? 16 : 8);
    g.blocks = 2 * a.pool.n_head;
    const uint32_t tiles = (g.page + kTileUnits - 1) / kTileUnits;
    // (a launch holds less than 2^32 threads)
    const uint32_t most = (uint32_t)((1ull << 23) / ((uint64_t)a.n_layer * tiles));
    if (most == 0) return hipErrorInvalidValue;
    return with_plan(a, ip, ib, [&](auto pa) {
        constexpr int INL = sizeof(pa.b) > 4 ? (int)sizeof(pa.b) : 0;
        hipError_t e = hipSuccess;
        for (uint32_t first = 0; first < a.n && e == hipSuccess; first += most)
            e = go(page_copy_kernel<INL>, (uint64_t)(a.n - first < most ? a.n - first : most) * a.n_layer * tiles, kCT, s,
                   LaunchTiming{}, a, g, tiles, first, pa);
        return e;
    });
}

}  // namespace ni
