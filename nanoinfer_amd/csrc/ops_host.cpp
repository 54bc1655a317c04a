// ops_host.cpp -- C ABI of the operators that need no cache handle: rotary
// positions over contiguous rows (ni_rotary_*) and the verification of drafted
// tokens (ni_verify_*).  Checks come before anything touches the device.
#include <hip/hip_runtime_api.h>

#include <algorithm>
#include <cmath>

#include "nanoinfer_kv.h"
#include "ops_plan.h"

using namespace ni;

namespace {

bool aligned(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

uint32_t type_bytes(uint32_t dtype) { return dtype == NI_F32 ? 4u : 2u; }

// Rows of `width` 4-byte values (aligned to them), `stride` apart.
struct Rows {
    const char* name;
    const void* p;
    int64_t stride, width;
};

// Whether n rows of a and n of b (where it is given) have a value in common.
bool share(const Rows& a, const Rows& b, uint32_t n) {
    if (!b.p) return false;
    typedef __int128 i128;
    const i128 from = ((i128)reinterpret_cast<uintptr_t>(a.p) - (i128)reinterpret_cast<uintptr_t>(b.p)) / 4;
    if (from >= (i128)(n - 1) * b.stride + b.width || from + (i128)(n - 1) * a.stride + a.width <= 0) return false;
    for (uint32_t i = 0; i < n; i++) {
        // The last row of b that begins at row i of a or before it, and the next.
        const i128 at = from + (i128)i * a.stride;
        const i128 j = b.stride > 0 && at > 0 ? std::min<i128>(at / b.stride, n - 1) : 0;
        for (i128 k = j; k <= j + 1 && k < n; k++)
            if (at < k * b.stride + b.width && at + a.width > k * b.stride) return true;
    }
    return false;
}

}  // namespace

extern "C" {

int ni_rotary_init(ni_rotary* r, uint32_t head_dim, const ni_rotary_opts* o) {
    if (!r || !o) return call_error(NI_ERR_BAD_ARG, "rotary and opts must not be NULL");
    const uint32_t rot = o->rot_dim ? o->rot_dim : head_dim;
    if (head_dim == 0 || head_dim % 2 != 0 || head_dim > 2 * NI_ROTARY_MAX_PAIRS)
        return call_error(NI_ERR_BAD_ARG, "head_dim %u must be even, 2..%u", head_dim, 2 * NI_ROTARY_MAX_PAIRS);
    if (rot % 2 != 0 || rot > head_dim)
        return call_error(NI_ERR_BAD_ARG, "rot_dim %u must be even and at most head_dim %u", rot, head_dim);
    if (o->interleaved > 1) return call_error(NI_ERR_BAD_ARG, "interleaved must be 0 or 1");
    if (!(o->base > 0) || !std::isfinite(o->base)) return call_error(NI_ERR_BAD_ARG, "base must be positive and finite");
    if (o->scaling > NI_ROTARY_YARN) return call_error(NI_ERR_BAD_ARG, "unknown scaling %u", o->scaling);
    if (o->scaling != NI_ROTARY_PLAIN && (!(o->factor >= 1) || !std::isfinite(o->factor)))
        return call_error(NI_ERR_BAD_ARG, "factor must be finite and at least 1");
    if (o->attn_scale < 0 || !std::isfinite(o->attn_scale))
        return call_error(NI_ERR_BAD_ARG, "attn_scale must be finite and not negative");
    // In 64-bit mantissas: a frequency of 53 bits would put angles 2^-25 turns off at
    // positions near 2^32.  These are (2 + 4) roundings of 2^-64 of f / 2 pi <= 0.16
    // turns off, a scaling's included, and half a unit of the table: below two units.
    const long double s = o->scaling == NI_ROTARY_PLAIN ? 1.L : o->factor;
    long double base = o->base, lo = 0.L, hi = 0.L, scale = 1.L;
    if (o->scaling == NI_ROTARY_NTK) {
        if (rot <= 2) return call_error(NI_ERR_BAD_ARG, "ntk scaling needs a rot_dim above 2");
        base *= std::pow(s, (long double)rot / (rot - 2));
    } else if (o->scaling == NI_ROTARY_YARN) {
        const long double fast = o->beta_fast > 0 ? o->beta_fast : 32., slow = o->beta_slow > 0 ? o->beta_slow : 1.;
        if (!(base > 1)) return call_error(NI_ERR_BAD_ARG, "yarn scaling needs a base above 1");
        if (o->orig_ctx == 0) return call_error(NI_ERR_BAD_ARG, "yarn scaling needs orig_ctx");
        if (!(fast >= slow)) return call_error(NI_ERR_BAD_ARG, "beta_fast must be at least beta_slow");
        // The pair that makes `turns` turns over the original context.
        auto pair = [&](long double turns) {
            return rot * std::log(o->orig_ctx / (turns * 2 * M_PIl)) / (2 * std::log(base));
        };
        lo = std::max(std::floor(pair(fast)), 0.L);
        hi = std::min(std::ceil(pair(slow)), (long double)rot - 1);
        if (s > 1) scale = 0.1L * std::log(s) + 1;
    }
    *r = ni_rotary{};
    r->head_dim = head_dim;
    r->rot_dim = rot;
    r->interleaved = o->interleaved;
    r->scale = (float)(o->attn_scale > 0 ? (long double)o->attn_scale : scale);
    for (uint32_t i = 0; i < rot / 2; i++) {
        long double f = std::pow(base, -2.L * i / rot);
        if (o->scaling == NI_ROTARY_LINEAR) f /= s;
        if (o->scaling == NI_ROTARY_YARN) {
            // Pairs that turn often keep their frequency, slow ones take the
            // stretched one, those between a mixture.
            const long double ramp = std::min(std::max((i - lo) / std::max(hi - lo, 0.001L), 0.L), 1.L);
            f = f / s * ramp + f * (1 - ramp);
        }
        const long double turns = f / (2 * M_PIl);
        r->turns[i] = (uint64_t)std::round(std::ldexp(turns - std::floor(turns), 64));  // 2^-64 of a turn: below 2^64
    }
    return NI_OK;
}

int ni_rotary_apply(const ni_rotary* r, uint32_t dtype, const void* x, int64_t x_row_stride, void* out,
                    int64_t out_row_stride, uint32_t n, uint32_t n_head, const int32_t* positions, uint32_t pos0,
                    ni_stream stream) {
    if (!r) return call_error(NI_ERR_BAD_ARG, "rotary is NULL");
    if (r->head_dim == 0 || r->head_dim % 2 != 0 || r->head_dim > 2 * NI_ROTARY_MAX_PAIRS || r->rot_dim == 0 ||
        r->rot_dim % 2 != 0 || r->rot_dim > r->head_dim || r->interleaved > 1)
        return call_error(NI_ERR_BAD_ARG, "rotary was not filled by ni_rotary_init");
    if (dtype > NI_BF16) return call_error(NI_ERR_BAD_ARG, "unknown type %u", dtype);
    if (n == 0 || n_head == 0) return NI_OK;
    const int64_t unit = 16 / type_bytes(dtype);
    const int64_t width = (int64_t)n_head * r->head_dim;
    if (!x || !out) return call_error(NI_ERR_BAD_ARG, "%s is NULL", x ? "out" : "x");
    if (!aligned(x, type_bytes(dtype)) || !aligned(out, type_bytes(dtype)) || x_row_stride < 0 || out_row_stride < 0)
        return call_error(NI_ERR_BAD_ARG, "x and out must be aligned to their type with non-negative row strides");
    if (n > 1 && out_row_stride < width)
        return call_error(NI_ERR_BAD_ARG, "out's rows overlap: the row stride must be at least %lld", (long long)width);
    if (out == x && n > 1 && x_row_stride != out_row_stride)
        return call_error(NI_ERR_BAD_ARG, "out may be x only with x's stride");
    if (!aligned(positions, 4)) return call_error(NI_ERR_BAD_ARG, "positions must be 4-byte aligned");
    // (a launch holds less than 2^32 threads, each of two values or eight)
    if ((unsigned __int128)n * width >= (1ull << 32)) return call_error(NI_ERR_BAD_ARG, "n * n_head * head_dim too large");
    RotaryLaunch a{};
    a.x = x;
    a.out = out;
    a.positions = positions;
    a.x_stride = x_row_stride;
    a.out_stride = out_row_stride;
    a.pos0 = pos0;
    a.n_rows = n;
    a.n_head = n_head;
    a.dtype = dtype;
    // Chunks of eight values, two or four heads' to a thread that turns by the same
    // angles, where every CU has many; pairs, a thread each, where the chunk's four
    // angles one after another are what takes the time (or on no 16-byte borders).  us
    // for pairs and for one, two and four heads: 64 x 12 x 64 f32 2.5, 3.2, 3.8, 4.8;
    // 512 x 12 x 64 2.7, 3.4, 3.9, 5.0; 4096 x 12 x 64 7.2, 6.2, 6.2, 7.3; bf16, 1024 x 40
    // x 128 10.5, 9.0, 7.6, 8.4; 2048 17.8, 14.2, 11.3, 11.4; 4095 31.7, 24.0, 17.8, 16.7.
    const uint64_t per_cu = (uint64_t)n * width / 8 / device_cus();
    a.wide = per_cu >= 256 && r->head_dim % 8 == 0 && r->rot_dim % 8 == 0 && aligned(x, 16) && aligned(out, 16) &&
             x_row_stride % unit == 0 && out_row_stride % unit == 0;
    a.heads_per = per_cu >= 4096 ? 4 : per_cu >= 2048 ? 2 : 1;
    const hipError_t e = launch_rotary(a, *r, (hipStream_t)stream);
    if (e != hipSuccess) return call_error(NI_ERR_HIP, "rotary launch failed: %s", hipGetErrorString(e));
    return NI_OK;
}

size_t ni_verify_workspace(uint32_t n_seq, uint32_t vocab) {
    return (size_t)n_seq * ((vocab + (uint64_t)kVerifyChunk - 1) / kVerifyChunk) * 2 * sizeof(double);
}

int ni_verify_drafts(uint32_t dtype, const void* target, int64_t target_seq_stride, int64_t target_row_stride,
                     const void* draft, int64_t draft_seq_stride, int64_t draft_row_stride, const int32_t* drafted,
                     int64_t drafted_stride, const int32_t* n_drafts, const float* accept_u, int64_t accept_stride,
                     const float* sample_u, uint32_t n_seq, uint32_t n_draft, uint32_t vocab, int32_t* accepted,
                     int32_t* tokens, int64_t tokens_stride, void* workspace, size_t workspace_bytes, ni_stream stream) {
    if (dtype > NI_BF16) return call_error(NI_ERR_BAD_ARG, "unknown type %u", dtype);
    if (n_seq == 0) return NI_OK;
    if (vocab == 0 || vocab > (1u << 30)) return call_error(NI_ERR_BAD_ARG, "vocab %u must be 1..2^30", vocab);
    if (n_seq > 65535) return call_error(NI_ERR_BAD_ARG, "%u sequences: at most 65535 a call", n_seq);
    if (n_draft > (1u << 20)) return call_error(NI_ERR_BAD_ARG, "n_draft %u too large", n_draft);
    const struct {
        const char* name;
        const void* p;
        bool needed;
        uintptr_t align;
        int64_t stride;
    } args[] = {{"target", target, true, type_bytes(dtype), std::min(target_seq_stride, target_row_stride)},
                {"draft", draft, false, type_bytes(dtype), draft ? std::min(draft_seq_stride, draft_row_stride) : 0},
                {"drafted", drafted, n_draft > 0, 4, n_draft ? drafted_stride : 0},
                {"n_drafts", n_drafts, false, 4, 0},
                {"accept_u", accept_u, n_draft > 0, 4, n_draft ? accept_stride : 0},
                {"sample_u", sample_u, true, 4, 0},
                {"accepted", accepted, true, 4, 0},
                {"tokens", tokens, true, 4, tokens_stride}};
    for (const auto& x : args) {
        if (x.needed && !x.p) return call_error(NI_ERR_BAD_ARG, "%s is NULL", x.name);
        if (!aligned(x.p, x.align)) return call_error(NI_ERR_BAD_ARG, "%s is not aligned to its type", x.name);
        if (x.stride < 0) return call_error(NI_ERR_BAD_ARG, "%s must have non-negative strides", x.name);
    }
    if (n_seq > 1 && tokens_stride < (int64_t)n_draft + 1)
        return call_error(NI_ERR_BAD_ARG, "tokens' rows overlap: the stride must be at least %u", n_draft + 1);
    const size_t need = ni_verify_workspace(n_seq, vocab);
    if (!workspace || !aligned(workspace, 16) || workspace_bytes < need)
        return call_error(NI_ERR_BAD_ARG, "workspace must be %zu bytes, 16-byte aligned", need);
    // (workgroups of one sequence read its drafts and numbers while another writes the answer)
    const Rows acc = {"accepted", accepted, 1, 1}, tok = {"tokens", tokens, tokens_stride, (int64_t)n_draft + 1};
    const Rows in[] = {{"n_drafts", n_drafts, 1, 1},
                       {"drafted", n_draft ? drafted : nullptr, drafted_stride, n_draft},
                       {"accept_u", n_draft ? accept_u : nullptr, accept_stride, n_draft},
                       {"sample_u", sample_u, 1, 1}};
    for (const Rows& x : in)
        for (const Rows& y : {acc, tok})
            if (share(y, x, n_seq)) return call_error(NI_ERR_BAD_ARG, "%s may not share memory with %s", y.name, x.name);
    if (share(tok, acc, n_seq)) return call_error(NI_ERR_BAD_ARG, "tokens may not share memory with accepted");
    VerifyLaunch a{};
    a.target = target;
    a.target_seq_stride = target_seq_stride;
    a.target_row_stride = target_row_stride;
    a.draft = draft;
    a.draft_seq_stride = draft_seq_stride;
    a.draft_row_stride = draft_row_stride;
    a.drafted = drafted;
    a.drafted_stride = drafted_stride;
    a.n_drafts = n_drafts;
    a.accept_u = accept_u;
    a.accept_stride = accept_stride;
    a.sample_u = sample_u;
    a.accepted = accepted;
    a.tokens = tokens;
    a.tokens_stride = tokens_stride;
    a.sums = static_cast<double*>(workspace);
    a.n_seq = n_seq;
    a.n_draft = n_draft;
    a.vocab = vocab;
    a.dtype = dtype;
    // As many chunks to a workgroup as leave every CU eight of them: the chain to the
    // first rejection is walked once for all, but a run of chunks takes longer.  us at
    // one, two and eight: 1 sequence of 50257 7.2, 7.9, 12.9; 64 of 131071 19.3, 18.5, 19.9;
    // 256 of 50257 23.6, 22.5, 22.3.
    const uint64_t chunks = (uint64_t)n_seq * ((vocab + (uint64_t)kVerifyChunk - 1) / kVerifyChunk);
    a.per = (uint32_t)std::min<uint64_t>(std::max<uint64_t>(chunks / (8ull * device_cus()), 1), 16);
    const hipError_t e = launch_verify(a, (hipStream_t)stream);
    if (e != hipSuccess) return call_error(NI_ERR_HIP, "verification launch failed: %s", hipGetErrorString(e));
    return NI_OK;
}

}  // extern "C"
