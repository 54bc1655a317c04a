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
#include "kv_device.h"
#include "ops_plan.h"

namespace ni {
namespace {

constexpr uint32_t kBT = 256;                   // threads of a scan
constexpr uint32_t kBE = kBeamChunk / kBT;      // entries a thread holds
constexpr uint32_t kGroupLanes = kBeamGroup / kBE;
static_assert(kBE == 8 && kGroupLanes == 16, "a group is a row of lanes");
constexpr float kLog2e = 1.44269504088896340736f;

// Whether anything of beam w of search b is read: it is alive, and goes on.
__device__ __forceinline__ bool is_finished(const BeamLaunch& a, uint32_t row) { return a.finished && a.finished[row] != 0; }

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
            for (int i = 0; i < (int)kBE / N; i++) w[i] = __builtin_nontemporal_load(reinterpret_cast<const V*>(row + v + N * i));
        } else {
#pragma unroll
            for (int i = 0; i < (int)kBE; i++) w[i / N][i % N] = v + i < vocab ? row[v + i] : (T)-INFINITY;
        }
    }
    __device__ __forceinline__ float at(int i) const { return (float)w[i / N][i % N]; }
};

// Workgroup (row, run of a.per chunks).
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
        const uint32_t v = chunk * kBeamChunk + threadIdx.x * kBE;
        if (chunk + 1 < chunk1) next.load(x, v + kBeamChunk, a.vocab);
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
        if (lane % kGroupLanes == 0 && v < a.vocab) groups[v / kBeamGroup] = top;
        cur = next;
    }
    // The workgroup's maximum and sum.
    float M = m;
    for (int off = 32; off > 0; off >>= 1) M = fmaxf(M, __shfl_xor(M, off));
    if (lane == 0) tops[threadIdx.x >> 6] = M;
    __syncthreads();
    M = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
    const float ref = fabsf(M) == INFINITY ? 0.f : M;
    double sum = s * (double)fast_exp2((m - ref) * kLog2e);
    for (int off = 32; off > 0; off >>= 1) sum += __shfl_xor(sum, off);
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

__device__ __forceinline__ Cand read_lane(const Cand& c, int l) {
    const uint64_t b = __builtin_bit_cast(uint64_t, c.total);
    const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)b, l), hi = __builtin_amdgcn_readlane((int)(uint32_t)(b >> 32), l);
    return Cand{__builtin_bit_cast(double, (uint64_t)hi << 32 | lo), (uint32_t)__builtin_amdgcn_readlane((int)c.index, l)};
}
// The lane before's value (lane 0: its own).
__device__ __forceinline__ uint32_t lane_before(uint32_t x) {
    return (uint32_t)__builtin_amdgcn_update_dpp((int)x, (int)x, 0x138, 0xf, 0xf, false);  // wave_shr:1
}

// A wave's best candidates so far, best first, one a lane (the first k are right).
struct Best {
    Cand c = {-INFINITY, 0xffffffffu};
    Cand last = {-INFINITY, 0xffffffffu};  // the k-th
    // Every lane offers one.
    __device__ __forceinline__ void offer(const Cand& x, uint32_t k) {
        uint64_t in = __ballot(x.total > -INFINITY && x.before(last.total, last.index));
        const uint32_t lane = threadIdx.x & 63u;
        while (in) {
            const int l = __builtin_amdgcn_readfirstlane(__ffsll((unsigned long long)in) - 1);
            in &= in - 1;
            const Cand y = read_lane(x, l);
            if (!y.before(last.total, last.index)) continue;
            const uint32_t at = (uint32_t)__popcll(__ballot(c.before(y.total, y.index)));
            const uint64_t bits = __builtin_bit_cast(uint64_t, c.total);
            const uint64_t up = (uint64_t)lane_before((uint32_t)(bits >> 32)) << 32 | lane_before((uint32_t)bits);
            const uint32_t up_i = lane_before(c.index);
            if (lane > at) {
                c.total = __builtin_bit_cast(double, up);
                c.index = up_i;
            } else if (lane == at) {
                c = y;
            }
            last = read_lane(c, (int)k - 1);
        }
    }
};

constexpr uint32_t kPT = 1024;          // threads of a pick
constexpr uint32_t kPW = kPT / 64;

// Where candidate sits among all waves' first k (those without a total behind the others): every thread of the
// workgroup takes part.  totals, indices: kPW * k entries; ranks as many counters, zeroed.
__device__ __forceinline__ void rank_all(const double* totals, const uint32_t* indices, uint32_t* ranks, uint32_t n) {
    // 2^j threads to a candidate, each against its share of the others
    uint32_t parts = 1;
    while (parts * 2 * n <= kPT) parts *= 2;
    const uint32_t i = threadIdx.x / parts, part = threadIdx.x - i * parts;
    if (i < n) {
        const Cand me = {totals[i], indices[i]};
        uint32_t before = 0;
        for (uint32_t j = part; j < n; j += parts) before += Cand{totals[j], indices[j]}.before(me.total, me.index) ? 1u : 0u;
        if (before) atomicAdd(&ranks[i], before);
    }
}

// One workgroup a search.
template <typename T>
__global__ __launch_bounds__(kPT) void beam_pick_kernel(const BeamLaunch a, const uint32_t chunks, const uint32_t runs) {
    __shared__ double offset[kBeamMax];           // score - normaliser: what a logit is added to
    __shared__ double totals[kPW * kBeamMax];
    __shared__ uint32_t indices[kPW * kBeamMax], ranks[kPW * kBeamMax];
    __shared__ uint32_t chosen[kBeamMax];         // groups, then (beam, token) of the answers
    __shared__ double best[kBeamMax];
    __shared__ uint8_t done[kBeamMax];
    const uint32_t b = blockIdx.x, W = a.n_beam, k = a.k, row0 = b * W;
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    for (uint32_t w = wave; w < W; w += kPW) {
        const float score = a.scores[row0 + w];
        const bool fin = is_finished(a, row0 + w);
        double off = -INFINITY;
        if (!fin && score > -INFINITY) {
            const BeamSum* p = a.sums + (uint64_t)(row0 + w) * chunks;
            float M = -INFINITY;
            for (uint32_t r = lane; r < runs; r += 64) M = fmaxf(M, p[r].top);
            for (int o = 32; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor(M, o));
            double S = 0.;
            if (fabsf(M) < INFINITY)
                for (uint32_t r = lane; r < runs; r += 64)
                    if (p[r].top > -INFINITY) S += (double)p[r].sum * exp((double)p[r].top - (double)M);
            for (int o = 32; o > 0; o >>= 1) S += __shfl_xor(S, o);
            if (fabsf(M) < INFINITY) off = (double)score - ((double)M + log(S));
        }
        if (lane == 0) {
            offset[w] = fin ? (double)score : off;
            done[w] = fin;
        }
    }
    for (uint32_t i = threadIdx.x; i < kPW * k; i += kPT) ranks[i] = 0;
    if (threadIdx.x < k) {
        chosen[threadIdx.x] = 0xffffffffu;
        best[threadIdx.x] = -INFINITY;
    }
    __syncthreads();
    // The groups.
    const uint32_t G = a.n_groups;
    {
        Best mine;
        // Of all beams one after another, eight loads at a time; a finished beam has one
        // candidate, in the pad token's group.
        const float* g = a.groups + (uint64_t)row0 * G;
        constexpr int U = 8;
        for (uint32_t i0 = threadIdx.x; i0 < W * G + threadIdx.x; i0 += U * kPT) {
            float x[U];
#pragma unroll
            for (int j = 0; j < U; j++) x[j] = i0 + j * kPT < W * G ? g[i0 + j * kPT] : -INFINITY;
#pragma unroll
            for (int j = 0; j < U; j++) {
                const uint32_t i = i0 + j * kPT, w = min(i / G, W - 1);
                const double off = offset[w];
                double t = off > -INFINITY ? off + (double)x[j] : -INFINITY;  // (the groups of others were not written)
                if (done[w]) t = i - w * G == a.pad / kBeamGroup ? off : -INFINITY;
                if (i >= W * G) t = -INFINITY;
                mine.offer(Cand{t, i}, k);
            }
        }
        if (lane < k) {
            totals[wave * k + lane] = mine.c.total;
            indices[wave * k + lane] = mine.c.index;
        }
    }
    __syncthreads();
    rank_all(totals, indices, ranks, kPW * k);
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < kPW * k; i += kPT) {
        if (ranks[i] < k && totals[i] > -INFINITY) chosen[ranks[i]] = indices[i];
        ranks[i] = 0;
    }
    __syncthreads();
    // Their entries.
    {
        Best mine;
        for (uint32_t c = wave; c < k; c += kPW) {
            const uint32_t gi = chosen[c];
            if (gi == 0xffffffffu) continue;
            const uint32_t w = gi / G, v0 = (gi - w * G) * kBeamGroup;
            const T* const x = static_cast<const T*>(a.logits) + (int64_t)b * a.search_stride + (int64_t)w * a.beam_stride;
            const double off = offset[w];
            T y[kBeamGroup / 64];
#pragma unroll
            for (uint32_t j = 0; j < kBeamGroup / 64; j++) {
                const uint32_t v = v0 + 64 * j + lane;
                y[j] = !done[w] && v < a.vocab ? x[v] : (T)-INFINITY;
            }
#pragma unroll
            for (uint32_t j = 0; j < kBeamGroup / 64; j++) {
                const uint32_t v = v0 + 64 * j + lane;
                double t = v < a.vocab ? off + (double)(float)y[j] : -INFINITY;
                if (done[w]) t = v == a.pad ? off : -INFINITY;
                mine.offer(Cand{t, w << kBeamTokenBits | v}, k);
            }
        }
        if (lane < k) {
            totals[wave * k + lane] = mine.c.total;
            indices[wave * k + lane] = mine.c.index;
        }
    }
    __syncthreads();
    if (threadIdx.x < k) chosen[threadIdx.x] = 0xffffffffu;
    rank_all(totals, indices, ranks, kPW * k);
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < kPW * k; i += kPT)
        if (ranks[i] < k && totals[i] > -INFINITY) {
            chosen[ranks[i]] = indices[i];
            best[ranks[i]] = totals[i];
        }
    __syncthreads();
    if (threadIdx.x < k) {
        const uint32_t c = chosen[threadIdx.x];
        const bool none = best[threadIdx.x] == -INFINITY;
        const uint64_t o = (uint64_t)b * k + threadIdx.x;
        a.out_scores[o] = (float)best[threadIdx.x];
        a.parents[o] = none ? -1 : (int32_t)(c >> kBeamTokenBits);
        a.tokens[o] = none ? -1 : (int32_t)(c & ((1u << kBeamTokenBits) - 1u));
    }
    if (a.out_history) {
        for (uint32_t i = wave; i < k; i += kPW) {
            const uint32_t c = chosen[i];
            const bool none = best[i] == -INFINITY;
            const int32_t* src = a.history + (int64_t)(row0 + (none ? 0 : c >> kBeamTokenBits)) * a.history_stride;
            int32_t* dst = a.out_history + (int64_t)((uint64_t)b * k + i) * a.out_history_stride;
            for (uint32_t j = lane; j < a.n_history; j += 64) dst[j] = none ? -1 : src[j];
            if (lane == 0) dst[a.n_history] = none ? -1 : (int32_t)(c & ((1u << kBeamTokenBits) - 1u));
        }
    }
}

template <typename T>
hipError_t beam_t(const BeamLaunch& a, hipStream_t s) {
    const uint32_t chunks = (a.vocab + kBeamChunk - 1) / kBeamChunk, runs = (chunks + a.per - 1) / a.per;
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
