// beam_kernels.hip -- gfx950 kernels of beam search's selection (ni_beam_select):
// the k best of score_w + log softmax(logits_w)_v over the beams w and the
// vocabulary v of each search.
//
//   beam_scan_kernel  every logit once: the sums of exp that normalise a row, and
//                     the largest logit of every kBeamGroup entries
//   beam_pick_kernel  the k groups with the best largest total, then the k best
//                     entries of those
//
// A row's totals lie in the order of its logits, so the k best entries lie in the k
// groups that are first by (largest total, lowest index): an entry of any other
// group has k entries before it.
//
// Totals are compared in 64 bits.  exp runs in f32 on differences from a lane's
// running maximum (1.6e-7 of a term that counts), eight terms are added in f32 (2^-21),
// all other sums and the logarithm run in 64 bits: with the maximum's few raises, 1e-7
// each, a normaliser is 2e-6 off at most, ~1e-8 as a rule.
#include <cfloat>
#include <type_traits>

#include "kv_device.h"
#include "ops_plan.h"

namespace ni {
namespace {

constexpr uint32_t kBT = 256;                   // threads of a scan
constexpr uint32_t kBE = kBeamChunk / kBT;      // entries a thread holds
constexpr uint32_t kGroupLanes = kBeamGroup / kBE;
static_assert(kBE == 8 && kGroupLanes == 16, "a group is a row of lanes");
constexpr float kLog2e = 1.44269504088896340736f;

// Whether a row's beam is finished: its logits are not read, it goes on with the pad token alone.
__device__ __forceinline__ bool is_finished(const BeamLaunch& a, uint32_t row) { return a.finished && a.finished[row] != 0; }

// Sum over groups of `lanes` lanes, a power of two up to 16.
__device__ __forceinline__ uint32_t lanes_sum(uint32_t x, uint32_t lanes) {
    const auto moved = [&](auto c) { return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, decltype(c)::value, 0xf, 0xf, false); };
    if (lanes >= 2) x += moved(std::integral_constant<int, 0xb1>{});
    if (lanes >= 4) x += moved(std::integral_constant<int, 0x4e>{});
    if (lanes >= 8) x += moved(std::integral_constant<int, 0x141>{});
    if (lanes >= 16) x += moved(std::integral_constant<int, 0x140>{});
    return x;
}
__device__ __forceinline__ uint32_t wave_sum(uint32_t x) {
    x = lanes_sum(x, 16);
    return (uint32_t)(__builtin_amdgcn_readlane((int)x, 0) + __builtin_amdgcn_readlane((int)x, 16) +
                      __builtin_amdgcn_readlane((int)x, 32) + __builtin_amdgcn_readlane((int)x, 48));
}
__device__ __forceinline__ float wave_top(float x) {
    x = fmaxf(x, dpp_move<0xb1>(x));
    x = fmaxf(x, dpp_move<0x4e>(x));
    x = fmaxf(x, dpp_move<0x141>(x));
    x = fmaxf(x, dpp_move<0x140>(x));
    return rows4_max(x);
}
template <int CTRL>
__device__ __forceinline__ double dpp_move64(double v) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)b, CTRL, 0xf, 0xf, false);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(b >> 32), CTRL, 0xf, 0xf, false);
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ double lane_of(double v, int l) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    return __builtin_bit_cast(double, (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(b >> 32), l) << 32 |
                                          (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)b, l));
}
__device__ __forceinline__ double wave_sum(double x) {
    x += dpp_move64<0xb1>(x);
    x += dpp_move64<0x4e>(x);
    x += dpp_move64<0x141>(x);
    x += dpp_move64<0x140>(x);
    return (lane_of(x, 0) + lane_of(x, 16)) + (lane_of(x, 32) + lane_of(x, 48));
}

// Eight neighbouring entries of a row from entry v on, those past the
// vocabulary -infinity.  Rows begin anywhere, so the wide loads ask for no more
// than an entry's alignment (which the memory system takes).
template <typename T>
struct Eight {
    static constexpr int N = 16 / sizeof(T);
    typedef T V __attribute__((ext_vector_type(N), aligned(sizeof(T))));
    V w[kBE / N];
    __device__ __forceinline__ void load(const T* row, uint32_t v, uint32_t vocab) {
        if (v + kBE <= vocab) {
#pragma unroll
            for (int i = 0; i < (int)kBE / N; i++) w[i] = *reinterpret_cast<const V*>(row + v + N * i);
        } else {
#pragma unroll
            for (int i = 0; i < (int)kBE; i++) w[i / N][i % N] = v + i < vocab ? row[v + i] : (T)-INFINITY;
        }
    }
    __device__ __forceinline__ float at(int i) const { return (float)w[i / N][i % N]; }
};

// Workgroup (row, run of a.per chunks).  Bound by the read: 64 x 8 rows of 131071 f32
// entries, 268 MB, 42 us, 6.4 TB/s; 16 x 6 rows of bf16, 20 MB, 8.0 us; four rows of 50257 3.0
// us, a launch.  A chunk's loads are in flight beside the sums of the one before.  (Non-temporal
// loads 52 us: logits that a product just wrote are partly in the caches.)
template <typename T>
__global__ __launch_bounds__(kBT) void beam_scan_kernel(const BeamLaunch a, const uint32_t chunks, const uint32_t runs) {
    __shared__ double sums[kBT / 64];
    __shared__ float tops[kBT / 64];
    const uint32_t row = blockIdx.x / runs, run = blockIdx.x - row * runs;
    const uint32_t b = row / a.n_beam, w = row - b * a.n_beam;
    if (is_finished(a, row) || !(a.scores[row] > -INFINITY)) return;
    const T* const x = static_cast<const T*>(a.logits) + (int64_t)b * a.search_stride + (int64_t)w * a.beam_stride;
    float* const groups = a.groups + (uint64_t)row * a.n_groups;
    const uint32_t chunk0 = run * a.per, chunk1 = min(chunk0 + a.per, chunks);
    const uint32_t lane = threadIdx.x & 63u;
    Eight<T> cur;
    cur.load(x, chunk0 * kBeamChunk + threadIdx.x * kBE, a.vocab);
    float m = -INFINITY;
    double s = 0.;
    for (uint32_t chunk = chunk0; chunk < chunk1; chunk++) {
        Eight<T> next = cur;
        const uint32_t p = chunk * kBeamChunk + threadIdx.x * kBE;
        if (chunk + 1 < chunk1) next.load(x, p + kBeamChunk, a.vocab);
        float y[kBE], top = -INFINITY;
#pragma unroll
        for (int i = 0; i < (int)kBE; i++) {
            y[i] = fmaxf(cur.at(i), -INFINITY);  // (a NaN is no candidate)
            top = fmaxf(top, y[i]);
        }
        const float mn = fmaxf(m, top);
        const float ref = mn == -INFINITY ? 0.f : mn;
        const double keep = (double)fast_exp2((m - ref) * kLog2e);
        m = mn;
        float e[kBE];
#pragma unroll
        for (int i = 0; i < (int)kBE; i++) e[i] = fast_exp2((y[i] - ref) * kLog2e);
        s = s * keep + (double)(((e[0] + e[1]) + (e[2] + e[3])) + ((e[4] + e[5]) + (e[6] + e[7])));
        top = fmaxf(top, dpp_move<0xb1>(top));
        top = fmaxf(top, dpp_move<0x4e>(top));
        top = fmaxf(top, dpp_move<0x141>(top));
        top = fmaxf(top, dpp_move<0x140>(top));
        if (lane % kGroupLanes == 0 && p / kBeamGroup < a.n_groups) groups[p / kBeamGroup] = top;
        cur = next;
    }
    // The workgroup's maximum and sum.
    float M = wave_top(m);
    if (lane == 0) tops[threadIdx.x >> 6] = M;
    __syncthreads();
    M = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
    const float ref = fabsf(M) == INFINITY ? 0.f : M;
    const double sum = wave_sum(s * (double)fast_exp2((m - ref) * kLog2e));
    if (lane == 0) sums[threadIdx.x >> 6] = sum;
    __syncthreads();
    if (threadIdx.x == 0) {
        BeamSum* p = a.sums + (uint64_t)row * chunks + run;
        p->top = M;
        p->sum = (float)((sums[0] + sums[1]) + (sums[2] + sums[3]));
    }
}

// A candidate: better by a higher total, then a lower index.
struct Cand {
    double total;
    uint32_t index;
    __device__ __forceinline__ bool before(double t, uint32_t i) const { return total > t || (total == t && index < i); }
};

constexpr uint32_t kPT = 1024;          // threads of a pick
constexpr uint32_t kPU = 8;             // candidates a thread holds at a time
constexpr uint32_t kList = 1024;        // candidates that are ranked at once
constexpr uint32_t kSetLanes = 16, kSets = kPT / kSetLanes;  // sets of candidates whose best are compared
static_assert(kPT * kPU == kBeamMax * kBeamGroup, "the entries of the chosen groups are looked at once");

struct Pick {
    double totals[kList];
    uint32_t indices[kList];
    __attribute__((aligned(16))) float tops[kSets];
    double best[kBeamMax];  // the answer so far, best first
    uint32_t best_index[kBeamMax];
    float bound;
    uint32_t n, counts[3];
};

// The first k of the n listed candidates into sh.best, in order: a candidate's place
// is the number of those before it.
__device__ __forceinline__ void rank_list(Pick& sh, uint32_t n, uint32_t k) {
    uint32_t parts = 1;  // threads to a candidate, each against its share of the others
    while (parts < 16 && parts * 2 * n <= kPT) parts *= 2;
    const uint32_t i = threadIdx.x / parts, part = threadIdx.x % parts;
    const Cand me = i < n ? Cand{sh.totals[i], sh.indices[i]} : Cand{0., 0u};
    uint32_t rank = 0;
    if (i < n)
        for (uint32_t j = part; j < n; j += parts) rank += Cand{sh.totals[j], sh.indices[j]}.before(me.total, me.index) ? 1u : 0u;
    rank = lanes_sum(rank, parts);
    if (i < n && part == 0 && rank < k) {
        sh.best[rank] = me.total;
        sh.best_index[rank] = me.index;
    }
}

// How many candidates of the workgroup are counted; turn: the number of the call.
__device__ __forceinline__ uint32_t count_all(Pick& sh, uint32_t mine, uint32_t turn) {
    const uint32_t at = turn % 3;  // (the counter of the call after next is cleared while this one's is read)
    if (threadIdx.x == 0) sh.counts[(turn + 1) % 3] = 0;
    mine = wave_sum(mine);
    if ((threadIdx.x & 63u) == 0 && mine) atomicAdd(&sh.counts[at], mine);
    __syncthreads();
    return sh.counts[at];
}

// Doubles as integers of the same order.
__device__ __forceinline__ uint64_t order_of(double x) {
    const uint64_t b = __builtin_bit_cast(uint64_t, x + 0.);  // (-0 as 0)
    return b >> 63 ? ~b : b | 1ull << 63;
}

// Candidates j of bit j of `in` into the list, as far as `room` goes; sh.n counts them all.
__device__ __forceinline__ void take(Pick& sh, const double (&t)[kPU], const uint32_t (&index)[kPU], uint32_t in, uint32_t room) {
    if (in == 0) return;
    // (few lanes have any: each adds for itself, which the compiler makes of an address that it cannot see to be one)
    uint32_t zero = 0;
    asm("" : "+v"(zero));
    uint32_t at = atomicAdd(&sh.n + zero, (uint32_t)__popc(in));
#pragma unroll
    for (uint32_t j = 0; j < kPU; j++)
        if (in >> j & 1u) {
            if (at < room) {
                sh.totals[at] = t[j];
                sh.indices[at] = index[j];
            }
            at++;
        }
}

// The first k of the workgroup's candidates into the list, behind the best so far, where
// more are left than it holds: the k-th total bit by bit, then the last index among its equals.
__device__ __forceinline__ void pick_equal(Pick& sh, const double (&t)[kPU], const uint32_t (&index)[kPU], uint32_t k,
                                           uint32_t have) {
    uint64_t key[kPU], kth = 0;
#pragma unroll
    for (uint32_t j = 0; j < kPU; j++) key[j] = t[j] > -INFINITY ? order_of(t[j]) : 0;
    if (threadIdx.x < 3) sh.counts[threadIdx.x] = 0;
    if (threadIdx.x == 0) sh.n = have;
    __syncthreads();
    uint32_t turn = 0;
    for (int bit = 63; bit >= 0; bit--) {
        const uint64_t trial = kth | 1ull << bit;
        uint32_t mine = 0;
#pragma unroll
        for (uint32_t j = 0; j < kPU; j++) mine += key[j] >= trial ? 1u : 0u;
        if (count_all(sh, mine, turn++) >= k) kth = trial;
    }
    uint32_t above = 0;
#pragma unroll
    for (uint32_t j = 0; j < kPU; j++) above += key[j] > kth ? 1u : 0u;
    const uint32_t equals = k - count_all(sh, above, turn++);
    uint32_t last = 0xffffffffu;  // the lowest index up to which there are as many
    for (int bit = 31; bit >= 0; bit--) {
        const uint32_t trial = last & ~(1u << bit);
        uint32_t mine = 0;
#pragma unroll
        for (uint32_t j = 0; j < kPU; j++) mine += key[j] == kth && index[j] <= trial ? 1u : 0u;
        if (count_all(sh, mine, turn++) >= equals) last = trial;
    }
    uint32_t in = 0;
#pragma unroll
    for (uint32_t j = 0; j < kPU; j++) in |= (key[j] > kth || (key[j] == kth && index[j] <= last) ? 1u : 0u) << j;
    take(sh, t, index, in, kList);
    __syncthreads();
}

// Bring the threads' candidates (-infinity: none) into the k best of sh.best, of which
// `have` are there; gives how many are then.  What lies below the k-th best of the
// bests of 64 sets of candidates is out; the few others are ranked with the best so
// far.  Every thread of the workgroup calls it.
__device__ __forceinline__ uint32_t pick_more(Pick& sh, const double (&t)[kPU], const uint32_t (&index)[kPU], uint32_t k,
                                              uint32_t have) {
    double high = t[0];
#pragma unroll
    for (uint32_t j = 1; j < kPU; j++) high = fmax(high, t[j]);
    float top = fminf((float)high, FLT_MAX);
    top -= fabsf(top) * 0x1p-23f;  // in f32, not above it
    top = fmaxf(top, dpp_move<0xb1>(top));
    top = fmaxf(top, dpp_move<0x4e>(top));
    top = fmaxf(top, dpp_move<0x141>(top));
    top = fmaxf(top, dpp_move<0x140>(top));
    static_assert(kSetLanes == 16 && kSets == 4 * kSetLanes, "a set is a row of lanes, each of which compares four");
    const uint32_t set = threadIdx.x / kSetLanes, part = threadIdx.x % kSetLanes;
    if (part == 0) sh.tops[set] = top;
    if (threadIdx.x == 0) sh.n = have;
    if (threadIdx.x < have) {  // the best so far begin the list
        sh.totals[threadIdx.x] = sh.best[threadIdx.x];
        sh.indices[threadIdx.x] = sh.best_index[threadIdx.x];
    }
    __syncthreads();
    uint32_t reach = 0;  // sets whose best is higher, and (16 bits up) no lower than this one's
    const float4 others = *reinterpret_cast<const float4*>(&sh.tops[4 * part]);
#pragma unroll
    for (int e = 0; e < 4; e++) {
        const float y = e == 0 ? others.x : e == 1 ? others.y : e == 2 ? others.z : others.w;
        reach += (y > top ? 1u : 0u) + (y >= top ? 1u << 16 : 0u);
    }
    reach = lanes_sum(reach, kSetLanes);
    // The k-th best: at least k candidates lie there or above.  (Equals write the same.)
    if (part == 0 && (reach & 0xffffu) < k && reach >> 16 >= k) sh.bound = top;
    __syncthreads();
    double bound = (double)sh.bound;
    if (have == k) bound = fmax(bound, sh.best[k - 1]);
    uint32_t in = 0;  // bit j: candidate j is not out
#pragma unroll
    for (uint32_t j = 0; j < kPU; j++) in |= (t[j] > -INFINITY && t[j] >= bound ? 1u : 0u) << j;
    take(sh, t, index, in, kList);
    __syncthreads();
    if (sh.n > kList) {
        __syncthreads();  // (everyone has seen it)
        pick_equal(sh, t, index, k, have);
    }
    const uint32_t n = sh.n;
    rank_list(sh, n, k);
    __syncthreads();
    return min(n, k);
}

// One workgroup a search: of 1800 groups 7.7 us, of 6100 9.8, of 8200 11.2, alike for any number
// of searches up to one a CU.  Bound by its chain of
// dependent steps: normalisers, bound over the groups, their ranks, the groups' entries from
// memory, bound and ranks again, histories.  Bounds by 64 sets' bests leave a few candidates
// more than k to rank; a choice of the best one by one took 31, 77 and 102 us.
template <typename T>
__global__ __launch_bounds__(kPT) void beam_pick_kernel(const BeamLaunch a, const uint32_t chunks, const uint32_t runs) {
    __shared__ Pick sh;
    __shared__ double offset[kBeamMax];    // score - normaliser: what a logit is added to
    __shared__ uint32_t chosen[kBeamMax];  // groups
    __shared__ uint8_t done[kBeamMax];
    const uint32_t b = blockIdx.x, W = a.n_beam, k = a.k, row0 = b * W, G = a.n_groups, all = W * G;
    const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // (G is a multiple of 64: the 64 groups of a wave are of one beam)
    auto beam_of = [&](uint32_t i) { return (uint32_t)(((uint64_t)(i / 64) * a.beam_magic) >> 32); };
    auto row_of = [&](uint32_t w) {
        return static_cast<const T*>(a.logits) + (int64_t)b * a.search_stride + (int64_t)w * a.beam_stride;
    };
    // The first groups' largest logits come while the normalisers are found.
    const float* const groups = a.groups + (uint64_t)row0 * G;
    float x[kPU];
    auto load = [&](uint32_t i0) {
#pragma unroll
        for (uint32_t j = 0; j < kPU; j++) {
            const uint32_t i = i0 + j * kPT + threadIdx.x;
            x[j] = i < all ? groups[i] : -INFINITY;
        }
    };
    load(0);
    for (uint32_t w = wave; w < W; w += kPT / 64) {
        const float score = a.scores[row0 + w];
        const bool fin = is_finished(a, row0 + w);
        double off = -INFINITY;
        if (!fin && score > -INFINITY) {
            const BeamSum* p = a.sums + (uint64_t)(row0 + w) * chunks;
            const BeamSum none = {-INFINITY, 0.f}, mine = lane < runs ? p[lane] : none;  // the first 64
            float M = mine.top;
            for (uint32_t r = lane + 64; r < runs; r += 64) M = fmaxf(M, p[r].top);
            M = wave_top(M);
            if (fabsf(M) < INFINITY) {
                auto part = [&](const BeamSum& x) {
                    return x.top > -INFINITY ? (double)x.sum * (double)fast_exp2((x.top - M) * kLog2e) : 0.;
                };
                double S = part(mine);
                for (uint32_t r = lane + 64; r < runs; r += 64) S += part(p[r]);
                off = (double)score - ((double)M + log(wave_sum(S)));
            }
        }
        if (lane == 0) {
            offset[w] = fin ? (double)score : off;
            done[w] = fin;
        }
    }
    __syncthreads();
    // The groups, kPT * kPU at a time, then the chosen ones' entries.  (One body for
    // both: the code is fetched anew for every launch.)
    uint32_t have = 0;
    for (uint32_t i0 = 0;; i0 += kPT * kPU) {
        const bool last = i0 >= all;
        double t[kPU];
        uint32_t index[kPU];
        if (!last) {
            if (i0 > 0) load(i0);
#pragma unroll
            for (uint32_t j = 0; j < kPU; j++) {
                const uint32_t at = i0 + j * kPT + wave * 64, i = at + lane;
                index[j] = i;
                t[j] = -INFINITY;
                if (at < all) {
                    const uint32_t w = beam_of(at);
                    const double off = offset[w];
                    // (what was not written -- groups past a row, of a beam that is finished or has no
                    // score -- may hold anything; a finished beam has one candidate, in its first)
                    double y = i - w * G < a.n_filled ? off + (double)x[j] : -INFINITY;
                    if (done[w]) y = i == w * G ? off : -INFINITY;
                    if (off > -INFINITY && y > -INFINITY) t[j] = y;
                }
            }
        } else {
            if (threadIdx.x < k) chosen[threadIdx.x] = threadIdx.x < have ? sh.best_index[threadIdx.x] : 0xffffffffu;
            __syncthreads();
            static_assert(kBeamGroup == 128, "two waves to a group");
            T y[kPU];
#pragma unroll
            for (uint32_t j = 0; j < kPU; j++) {
                const uint32_t c = (j * kPT / 64 + wave) / 2, e = wave % 2 * 64 + lane;
                y[j] = (T)-INFINITY;
                index[j] = 0xffffffffu;
                if (c < have) {
                    const uint32_t g = __builtin_amdgcn_readfirstlane(chosen[c]), w = beam_of(g);
                    const uint32_t v = (g - w * G) * kBeamGroup + e;
                    const bool fin = done[w], in = !fin && v < a.vocab;
                    if (in) y[j] = row_of(w)[v];
                    if (in || (fin && e == 0)) index[j] = w << kBeamTokenBits | (fin ? a.pad : v);
                }
            }
#pragma unroll
            for (uint32_t j = 0; j < kPU; j++) {
                const uint32_t w = index[j] >> kBeamTokenBits;
                double z = -INFINITY;
                if (index[j] != 0xffffffffu) z = done[w] ? offset[w] : offset[w] + (double)(float)y[j];
                t[j] = z > -INFINITY ? z : -INFINITY;
            }
            have = 0;
        }
        have = pick_more(sh, t, index, k, have);
        if (last) break;
    }
    if (threadIdx.x < k) {
        const bool none = threadIdx.x >= have;
        const uint32_t c = sh.best_index[threadIdx.x];
        const uint64_t o = (uint64_t)b * k + threadIdx.x;
        a.out_scores[o] = none ? -INFINITY : (float)sh.best[threadIdx.x];
        a.parents[o] = none ? -1 : (int32_t)(c >> kBeamTokenBits);
        a.tokens[o] = none ? -1 : (int32_t)(c & ((1u << kBeamTokenBits) - 1u));
    }
    if (a.out_history) {
        for (uint32_t i = wave; i < k; i += kPT / 64) {
            const bool none = i >= have;
            const uint32_t c = none ? 0 : sh.best_index[i];
            const int32_t* src = a.history + (int64_t)(row0 + (c >> kBeamTokenBits)) * a.history_stride;
            int32_t* dst = a.out_history + (int64_t)((uint64_t)b * k + i) * a.out_history_stride;
            for (uint32_t j = lane; j < a.n_history; j += 64) dst[j] = none ? -1 : src[j];
            if (lane == 0) dst[a.n_history] = none ? -1 : (int32_t)(c & ((1u << kBeamTokenBits) - 1u));
        }
    }
}

template <typename T>
hipError_t beam_t(const BeamLaunch& a, hipStream_t s) {
    const uint32_t chunks = beam_chunks(a.vocab), runs = (chunks + a.per - 1) / a.per;
    hipLaunchKernelGGL(beam_scan_kernel<T>, dim3(a.n_search * a.n_beam * runs), dim3(kBT), 0, s, a, chunks, runs);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(beam_pick_kernel<T>, dim3(a.n_search), dim3(kPT), 0, s, a, chunks, runs);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_beam(const BeamLaunch& a, hipStream_t s) {
    switch (a.dtype) {
        case NI_F32: return beam_t<float>(a, s);
        case NI_F16: return beam_t<_Float16>(a, s);
        case NI_BF16: return beam_t<__bf16>(a, s);
        default: return hipErrorInvalidValue;
    }
}

}  // namespace ni
