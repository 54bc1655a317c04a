// verify_kernels.hip -- gfx950 kernels of the verification of drafted tokens
// against a target model's probabilities (ni_verify_drafts).
//
//   verify_sums_kernel  each sequence's first rejection, and the sums of
//                       kVerifyChunk entries of the row to draw from
//   verify_draw_kernel  the entry at which the running sum passes u times the
//                       whole
//
// Draft i (token t) stays while u_i q_i(t) < p_i(t).  u, p and q are f32 or
// narrower, so u q is exact in 64 bits and the comparison is the definition's
// own.  The sums run in 64 bits: at 2^17 entries they are ~1e-14 of the whole
// off, and the drawn entry is that of any other 64-bit order unless u lands
// that near a border.
#include "kv_device.h"
#include "ops_plan.h"

namespace ni {
namespace {

constexpr uint32_t kVT = 256;                    // threads
constexpr uint32_t kVE = kVerifyChunk / kVT;      // entries a thread holds

// A probability of row `p` (f32, f16 or bf16).
template <typename T>
__device__ __forceinline__ double prob(const void* p, int64_t i) {
    return (double)static_cast<const T*>(p)[i];
}

// A weight to draw by: negative values and NaN weigh nothing.
__device__ __forceinline__ double weight(double x) { return x > 0. ? x : 0.; }

// Drafts of sequence b that are looked at.
__device__ __forceinline__ uint32_t drafts_of(const VerifyLaunch& a, uint32_t b) {
    if (!a.n_drafts) return a.n_draft;
    const int32_t n = a.n_drafts[b];
    return n < 0 ? 0u : min((uint32_t)n, a.n_draft);
}

// Drafts of sequence b accepted: those before the first rejection.  Every
// lane of the wave gets the answer.
template <typename T>
__device__ __forceinline__ uint32_t accepted_of(const VerifyLaunch& a, uint32_t b, uint32_t n) {
    const uint32_t lane = threadIdx.x & 63u;
    for (uint32_t i0 = 0; i0 < n; i0 += 64) {
        const uint32_t i = i0 + lane;
        bool ok = true;
        if (i < n) {
            const int32_t t = a.drafted[(int64_t)b * a.drafted_stride + i];
            ok = t >= 0 && (uint32_t)t < a.vocab;  // a token outside the vocabulary is rejected
            if (ok) {
                const double p = prob<T>(a.target, (int64_t)b * a.target_seq_stride + (int64_t)i * a.target_row_stride + t);
                const double q =
                    a.draft ? prob<T>(a.draft, (int64_t)b * a.draft_seq_stride + (int64_t)i * a.draft_row_stride + t) : 1.;
                ok = (double)a.accept_u[(int64_t)b * a.accept_stride + i] * q < p;
            }
        }
        const uint64_t no = __ballot(!ok);
        if (no) return i0 + (uint32_t)__ffsll((unsigned long long)no) - 1u;
    }
    return n;
}

// The row to draw from: the target's row `at`, less the drafter's where draft
// `at` was rejected.
struct Row {
    int64_t p, q;    // element offsets of the two rows
    int32_t token;   // the rejected token
    bool rejected;
};
__device__ __forceinline__ Row row_of(const VerifyLaunch& a, uint32_t b, uint32_t at, uint32_t n) {
    Row r;
    r.rejected = at < n;
    r.p = (int64_t)b * a.target_seq_stride + (int64_t)at * a.target_row_stride;
    r.q = r.rejected && a.draft ? (int64_t)b * a.draft_seq_stride + (int64_t)at * a.draft_row_stride : 0;
    r.token = r.rejected ? a.drafted[(int64_t)b * a.drafted_stride + at] : -1;
    return r;
}
// What is left of the target's probability p of entry v.
template <typename T>
__device__ __forceinline__ double left(const VerifyLaunch& a, const Row& r, uint32_t v, double p) {
    if (!r.rejected) return weight(p);
    if (a.draft) return weight(p - prob<T>(a.draft, r.q + v));
    return (int32_t)v == r.token ? 0. : weight(p);
}

__device__ __forceinline__ double wave_sum(double x) {
    for (int off = 32; off > 0; off >>= 1) x += __shfl_xor(x, off);
    return x;
}

// Workgroup (chunk, sequence).
template <typename T>
__global__ __launch_bounds__(kVT) void verify_sums_kernel(const VerifyLaunch a) {
    __shared__ double sh[2][kVT / 64];
    const uint32_t b = blockIdx.y, chunk = blockIdx.x;
    const uint32_t n = drafts_of(a, b);
    const uint32_t at = accepted_of<T>(a, b, n);
    if (chunk == 0) {
        if (threadIdx.x == 0) a.accepted[b] = (int32_t)at;
        for (uint32_t i = threadIdx.x; i <= a.n_draft; i += kVT)
            if (i != at) a.tokens[(int64_t)b * a.tokens_stride + i] = i < at ? a.drafted[(int64_t)b * a.drafted_stride + i] : -1;
    }
    const Row r = row_of(a, b, at, n);
    double sl = 0., sp = 0.;
#pragma unroll
    for (uint32_t e = 0; e < kVE; e++) {
        const uint32_t v = chunk * kVerifyChunk + e * kVT + threadIdx.x;
        if (v < a.vocab) {
            const double p = prob<T>(a.target, r.p + v);
            sl += left<T>(a, r, v, p);
            sp += weight(p);
        }
    }
    sl = wave_sum(sl);
    sp = wave_sum(sp);
    if ((threadIdx.x & 63) == 0) {
        sh[0][threadIdx.x >> 6] = sl;
        sh[1][threadIdx.x >> 6] = sp;
    }
    __syncthreads();
    if (threadIdx.x < 2) {
        const double* x = sh[threadIdx.x];
        a.sums[((uint64_t)b * gridDim.x + chunk) * 2 + threadIdx.x] = (x[0] + x[1]) + (x[2] + x[3]);
    }
}

// Inclusive running sum over the workgroup's threads, and the whole.
__device__ __forceinline__ double block_scan(double x, double* sh, double& whole) {
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    for (int off = 1; off < 64; off <<= 1) {
        const double y = __shfl_up(x, off);
        if (lane >= (uint32_t)off) x += y;
    }
    __syncthreads();
    if (lane == 63) sh[wave] = x;
    __syncthreads();
    double before = 0.;
    whole = 0.;
    for (uint32_t w = 0; w < kVT / 64; w++) {
        if (w < wave) before += sh[w];
        whole += sh[w];
    }
    return before + x;
}

// One workgroup a sequence: the chunk in which the running sum passes u times
// the whole, then the entry.  Where rounding leaves no entry past it, the last
// with any weight; -1 where none has.
template <typename T>
__global__ __launch_bounds__(kVT) void verify_draw_kernel(const VerifyLaunch a, const uint32_t chunks) {
    __shared__ double sh[kVT / 64];
    __shared__ uint32_t first, last;  // the chunk (then the entry) that passes, and the last with weight, plus one
    const uint32_t b = blockIdx.x;
    const uint32_t n = drafts_of(a, b);
    const uint32_t at = (uint32_t)a.accepted[b];
    const Row r = row_of(a, b, at, n);
    const double* sums = a.sums + (uint64_t)b * chunks * 2;
    double whole_left = 0., whole_p = 0.;
    for (uint32_t c = threadIdx.x; c < chunks; c += kVT) {
        whole_left += sums[2 * c];
        whole_p += sums[2 * c + 1];
    }
    double x;
    block_scan(whole_left, sh, x);
    whole_left = x;
    block_scan(whole_p, sh, x);
    whole_p = x;
    // Nothing is left (the target's row lies under the drafter's): the row itself.
    const bool rest = r.rejected && whole_left > 0.;
    const double u = (double)a.sample_u[b];
    const double pass = u * (rest ? whole_left : whole_p);
    if (threadIdx.x == 0) {
        first = 0xffffffffu;
        last = 0;
    }
    __syncthreads();
    double base = 0.;
    for (uint32_t c0 = 0; c0 < chunks; c0 += kVT) {
        const uint32_t c = c0 + threadIdx.x;
        const double w = c < chunks ? sums[2 * c + (rest ? 0 : 1)] : 0.;
        double whole;
        const double run = base + block_scan(w, sh, whole);
        if (w > 0.) {
            if (run > pass) atomicMin(&first, c);
            atomicMax(&last, c + 1);
        }
        base += whole;
    }
    __syncthreads();
    if (last == 0) {
        if (threadIdx.x == 0) a.tokens[(int64_t)b * a.tokens_stride + at] = -1;
        return;
    }
    const uint32_t chunk = min(first, last - 1);
    // The sum of the chunks before it.
    double before = 0.;
    for (uint32_t c = threadIdx.x; c < chunk; c += kVT) before += sums[2 * c + (rest ? 0 : 1)];
    block_scan(before, sh, x);
    before = x;
    __syncthreads();
    if (threadIdx.x == 0) {
        first = 0xffffffffu;
        last = 0;
    }
    __syncthreads();
    double w[kVE], sum = 0.;
    const uint32_t v0 = chunk * kVerifyChunk + threadIdx.x * kVE;
#pragma unroll
    for (uint32_t e = 0; e < kVE; e++) {
        w[e] = 0.;
        if (v0 + e < a.vocab) {
            const double p = prob<T>(a.target, r.p + v0 + e);
            w[e] = rest ? left<T>(a, r, v0 + e, p) : weight(p);
        }
        sum += w[e];
    }
    double run = before + block_scan(sum, sh, x) - sum;
#pragma unroll
    for (uint32_t e = 0; e < kVE; e++) {
        run += w[e];
        if (w[e] > 0.) {
            if (run > pass) atomicMin(&first, v0 + e);
            atomicMax(&last, v0 + e + 1);
        }
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        // (the chunk's own sum is positive, so some entry has weight)
        a.tokens[(int64_t)b * a.tokens_stride + at] = first != 0xffffffffu ? (int32_t)first : (int32_t)last - 1;
    }
}

template <typename T>
hipError_t verify_t(const VerifyLaunch& a, hipStream_t s) {
    const uint32_t chunks = (a.vocab + kVerifyChunk - 1) / kVerifyChunk;
    hipLaunchKernelGGL(verify_sums_kernel<T>, dim3(chunks, a.n_seq), dim3(kVT), 0, s, a);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(verify_draw_kernel<T>, dim3(a.n_seq), dim3(kVT), 0, s, a, chunks);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_verify(const VerifyLaunch& a, hipStream_t s) {
    switch (a.dtype) {
        case NI_F32: return verify_t<float>(a, s);
        case NI_F16: return verify_t<_Float16>(a, s);
        case NI_BF16: return verify_t<__bf16>(a, s);
        default: return hipErrorInvalidValue;
    }
}

}  // namespace ni
