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
static_assert(kVE == 8, "a thread's entries come in 16-byte loads");

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
    r.token = r.rejected && !a.draft ? a.drafted[(int64_t)b * a.drafted_stride + at] : -1;
    return r;
}

// Eight neighbouring entries of a row from entry v on, those past the
// vocabulary 0.  Rows begin anywhere, so the wide loads ask for no more than an
// entry's alignment (which the memory system takes).
template <typename T>
__device__ __forceinline__ void load8(const void* base, int64_t row, uint32_t v, uint32_t vocab, float (&x)[kVE]) {
    const T* p = static_cast<const T*>(base) + row + v;
    if (v + kVE <= vocab) {
        typedef T V __attribute__((ext_vector_type(16 / sizeof(T)), aligned(sizeof(T))));
        constexpr int N = 16 / sizeof(T);
        V w[kVE / N];
#pragma unroll
        for (int i = 0; i < (int)kVE / N; i++) w[i] = *reinterpret_cast<const V*>(p + N * i);
#pragma unroll
        for (int i = 0; i < (int)kVE; i++) x[i] = (float)w[i / N][i % N];
    } else {
#pragma unroll
        for (int i = 0; i < (int)kVE; i++) x[i] = v + i < vocab ? (float)p[i] : 0.f;
    }
}
// Entries v .. v + 7 of row r: the target's weights wp and what is left of them, wl.
template <typename T>
__device__ __forceinline__ void weights8(const VerifyLaunch& a, const Row& r, uint32_t v, double (&wl)[kVE],
                                         double (&wp)[kVE]) {
    float p[kVE], q[kVE];
    load8<T>(a.target, r.p, v, a.vocab, p);
    const bool less = r.rejected && a.draft;
    if (less) load8<T>(a.draft, r.q, v, a.vocab, q);
#pragma unroll
    for (int i = 0; i < (int)kVE; i++) {
        wp[i] = weight((double)p[i]);
        wl[i] = less ? weight((double)p[i] - (double)q[i]) : (int32_t)(v + i) == r.token ? 0. : wp[i];
    }
}

__device__ __forceinline__ double wave_sum(double x) {
    for (int off = 32; off > 0; off >>= 1) x += __shfl_xor(x, off);
    return x;
}

// Workgroup (run of a.per chunks, sequence): few enough that the chain to the
// first rejection (draft count, token, probabilities: three loads one after
// another) is walked once per run.  64 sequences of 131071 f32, a third of which end on
// a rejection and read the drafter's row too, 45 MB: 11 us (4.1 TB/s; a chunk's loads
// wait for the sums of the one before); one of 50257 3.6.
template <typename T>
__global__ __launch_bounds__(kVT) void verify_sums_kernel(const VerifyLaunch a, const uint32_t chunks) {
    __shared__ double2 sh[2][kVT / 64];
    const uint32_t b = blockIdx.y, chunk0 = blockIdx.x * a.per, chunk1 = min(chunk0 + a.per, chunks);
    const uint32_t n = drafts_of(a, b);
    const uint32_t at = accepted_of<T>(a, b, n);
    if (chunk0 == 0) {
        if (threadIdx.x == 0) a.accepted[b] = (int32_t)at;
        for (uint32_t i = threadIdx.x; i <= a.n_draft; i += kVT)
            if (i != at) a.tokens[(int64_t)b * a.tokens_stride + i] = i < at ? a.drafted[(int64_t)b * a.drafted_stride + i] : -1;
    }
    const Row r = row_of(a, b, at, n);
    for (uint32_t chunk = chunk0; chunk < chunk1; chunk++) {
        double wl[kVE], wp[kVE];
        weights8<T>(a, r, chunk * kVerifyChunk + threadIdx.x * kVE, wl, wp);
        double sl = ((wl[0] + wl[1]) + (wl[2] + wl[3])) + ((wl[4] + wl[5]) + (wl[6] + wl[7]));
        double sp = ((wp[0] + wp[1]) + (wp[2] + wp[3])) + ((wp[4] + wp[5]) + (wp[6] + wp[7]));
        sl = wave_sum(sl);
        sp = wave_sum(sp);
        double2* x = sh[chunk & 1];  // (the other half may still be read)
        if ((threadIdx.x & 63) == 0) x[threadIdx.x >> 6] = double2{sl, sp};
        __syncthreads();
        if (threadIdx.x == 0)
            reinterpret_cast<double2*>(a.sums)[(uint64_t)b * chunks + chunk] =
                double2{(x[0].x + x[1].x) + (x[2].x + x[3].x), (x[0].y + x[1].y) + (x[2].y + x[3].y)};
    }
}

// Inclusive running sum over the lanes of a wave.
__device__ __forceinline__ double wave_scan(double x) {
    const uint32_t lane = threadIdx.x & 63u;
    for (int off = 1; off < 64; off <<= 1) {
        const double y = __shfl_up(x, off);
        if (lane >= (uint32_t)off) x += y;
    }
    return x;
}

// One workgroup a sequence: the chunk in which the running sum passes u times
// the whole (every wave finds it by itself, 64 chunks at a time), then the
// entry.  Where rounding leaves no entry past it, the last with any weight; -1
// where none has.  4-5 us: the sums, then the chunk, one load after another.
template <typename T>
__global__ __launch_bounds__(kVT) void verify_draw_kernel(const VerifyLaunch a, const uint32_t chunks) {
    __shared__ double wave_sums[kVT / 64];
    __shared__ int32_t firsts[kVT / 64], lasts[kVT / 64];
    const uint32_t b = blockIdx.x, lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    const uint32_t n = drafts_of(a, b);
    const uint32_t at = (uint32_t)a.accepted[b];
    const double u = (double)a.sample_u[b];
    const double2* sums = reinterpret_cast<const double2*>(a.sums) + (uint64_t)b * chunks;
    const double2 mine = lane < chunks ? sums[lane] : double2{0., 0.};  // the first 64 chunks
    const Row r = row_of(a, b, at, n);
    double whole_left = mine.x, whole_p = mine.y;
    for (uint32_t c = lane + 64; c < chunks; c += 64) {
        whole_left += sums[c].x;
        whole_p += sums[c].y;
    }
    whole_left = wave_sum(whole_left);
    whole_p = wave_sum(whole_p);
    // Nothing is left (the target's row lies under the drafter's): the row itself.
    const bool rest = r.rejected && whole_left > 0.;
    const double pass = u * (rest ? whole_left : whole_p);
    uint32_t chunk = 0xffffffffu, last = 0xffffffffu;  // that passes; the last with weight
    double before = 0., before_last = 0., base = 0.;   // the sums ahead of them
    for (uint32_t c0 = 0; c0 < chunks && chunk == 0xffffffffu; c0 += 64) {
        const uint32_t c = c0 + lane;
        const double2 s = c0 == 0 ? mine : c < chunks ? sums[c] : double2{0., 0.};
        const double w = rest ? s.x : s.y;
        const double run = base + wave_scan(w);
        const uint64_t has = __ballot(w > 0.), over = __ballot(w > 0. && run > pass);
        double ahead = __shfl_up(run, 1);
        if (lane == 0) ahead = base;
        if (over) {
            const int l = __ffsll((unsigned long long)over) - 1;
            chunk = c0 + l;
            before = __shfl(ahead, l);
        } else if (has) {
            const int l = 63 - __clzll((long long)has);
            last = c0 + l;
            before_last = __shfl(ahead, l);
        }
        base = __shfl(run, 63);
    }
    if (chunk == 0xffffffffu) {
        chunk = last;
        before = before_last;
    }
    if (chunk == 0xffffffffu) {
        if (threadIdx.x == 0) a.tokens[(int64_t)b * a.tokens_stride + at] = -1;
        return;
    }
    double wl[kVE], wp[kVE];
    const uint32_t v0 = chunk * kVerifyChunk + threadIdx.x * kVE;
    weights8<T>(a, r, v0, wl, wp);
    double run[kVE], sum = 0.;  // running sums of the thread's own entries
#pragma unroll
    for (int i = 0; i < (int)kVE; i++) {
        if (!rest) wl[i] = wp[i];
        sum += wl[i];
        run[i] = sum;
    }
    const double upto = wave_scan(sum);
    if (lane == 63) wave_sums[wave] = upto;
    __syncthreads();
    for (uint32_t w = 0; w < wave; w++) before += wave_sums[w];
    double ahead = __shfl_up(upto, 1);
    before += lane == 0 ? 0. : ahead;
    int32_t first_e = -1, last_e = -1;
#pragma unroll
    for (int i = (int)kVE - 1; i >= 0; i--)
        if (wl[i] > 0.) {
            if (before + run[i] > pass) first_e = (int32_t)v0 + i;
            if (last_e < 0) last_e = (int32_t)v0 + i;
        }
    const uint64_t over = __ballot(first_e >= 0), has = __ballot(last_e >= 0);
    const int f = over ? __shfl(first_e, __ffsll((unsigned long long)over) - 1) : -1;
    const int l = has ? __shfl(last_e, 63 - __clzll((long long)has)) : -1;
    if (lane == 0) {
        firsts[wave] = f;
        lasts[wave] = l;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        int32_t t = -1;
        for (int w = 0; w < (int)kVT / 64 && t < 0; w++) t = firsts[w];
        for (int w = (int)kVT / 64 - 1; w >= 0 && t < 0; w--) t = lasts[w];
        a.tokens[(int64_t)b * a.tokens_stride + at] = t;
    }
}

template <typename T>
hipError_t verify_t(const VerifyLaunch& a, hipStream_t s) {
    const uint32_t chunks = (a.vocab + kVerifyChunk - 1) / kVerifyChunk;
    hipLaunchKernelGGL(verify_sums_kernel<T>, dim3((chunks + a.per - 1) / a.per, a.n_seq), dim3(kVT), 0, s, a, chunks);
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
