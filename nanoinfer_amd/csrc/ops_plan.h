// ops_plan.h -- what the host hands to the kernels of the rotary, shared-prefix
// and verification operators (rotary_kernels.hip, prefix_kernels.hip,
// verify_kernels.hip).  The host checks every index and size before it
// launches; the kernels check what only the device can see (token ids, draft
// counts).
#pragma once

#include "kv_plan.h"
#include "nanoinfer_kv.h"

namespace ni {

// ---------------------------------------------------------------- rotary

// Contiguous rows (ni_rotary_apply).
struct RotaryLaunch {
    const void* x;
    void* out;
    const int32_t* positions;  // device, or null: row i is at pos0 + i
    int64_t x_stride, out_stride;
    uint32_t pos0;
    uint32_t n_rows;
    uint32_t n_head;
    uint32_t dtype;      // NI_F32, NI_F16, NI_BF16
    uint32_t heads_per;  // heads one thread rotates with the same cosines
    uint32_t wide;       // chunks of 8 values: sizes and addresses are multiples of 8 values
};
hipError_t launch_rotary(const RotaryLaunch& a, const ni_rotary& r, hipStream_t s);

// Pairs of a head in the cache (head_dim 64 or 128), passed with the launch.
constexpr uint32_t kCachePairs = 64;
struct CacheRotary {
    uint32_t rot_dim;
    uint32_t interleaved;
    float scale;
    uint32_t pad;
    uint64_t turns[kCachePairs];
};

// The append with the rotation on the way (ni_kv_append_rotary).  Entry i: where
// input row i goes.  Eight bytes, so that up to 256 rows travel in the smallest
// argument block (160 rows in 16-byte entries: 8.4 us of host time a call, 7.0).
struct RotaryEntry {
    uint32_t pos;    // position it is rotated to
    uint32_t place;  // page * kPage + slot
};
constexpr uint32_t kMaxRotaryPages = 0xffffffffu / kPage;
struct AppendRotaryLaunch {
    PoolGeom pool;
    const float* q;  // null: no queries
    const float* k;
    const float* v;
    float* q_out;
    int64_t q_row_stride, q_layer_stride;
    int64_t q_out_row_stride, q_out_layer_stride;
    int64_t row_stride, layer_stride;  // k and v
    const uint8_t* plan;
    uint32_t off_entries;
    uint32_t n_rows;
    uint32_t layer0;
    uint32_t n_lay;
    uint32_t n_q_head;  // 0: no queries
    uint32_t parts;     // workgroups of a (layer, row) ...
    uint32_t share;     // ... of this many chunks of 8 values each (a multiple of 256)
};
hipError_t launch_append_rotary(const AppendRotaryLaunch& a, const CacheRotary& r, const void* inline_plan,
                                uint32_t inline_bytes, hipStream_t s, const LaunchTiming& t = {});

// ------------------------------------------------ shared-prefix attention

// Queries travel as slots: the G = n_q_head / n_head query heads that read one
// cache head, row by row: slot s of a run of rows is head s % G of row s / G.
constexpr uint32_t kSlotTile = 16;            // slots of an item
constexpr uint32_t kWideSlots = 32;           // slots of one wave of a wide item ...
constexpr uint32_t kWideWavesMax = 4;         // ... of this many waves at most
// Groups of waves that share a wide workgroup's keys.
constexpr int wide_groups(int head_dim, int waves) { return head_dim == 64 ? (waves <= 2 ? 4 : 2) : 2; }
constexpr uint32_t kWholePos = 0x7fffffffu;   // PrefixItem::pos0 of a prefix: every slot sees every key

// One work item: slots slot0 .. slot0 + ns - 1 of the run of rows at row0 over
// keys [kv_begin, kv_end) of one page list.  Slot s sees keys <= pos0 + s / G.
// An item whose part0 is kNoSlot holds all its slots' own keys: it joins the
// n_pre partials of their prefix (those of slot s at pre0 + s + j * pre_stride,
// written by an earlier launch) and writes their outputs.
struct PrefixItem {
    uint32_t tab;       // the page list, in the plan's table
    uint32_t row0;
    uint32_t slot0;
    uint32_t ns;
    uint32_t pos0;
    uint32_t kv_begin;  // a multiple of kPage
    uint32_t kv_end;
    uint32_t part0;     // partial of the first slot, or kNoSlot
    uint32_t pre0, pre_stride, n_pre;
    uint32_t pad;
};

// The partials of one row's slots: n_own of its own keys' partitions, n_pre
// of the prefix's, each `stride` partials from the one before.
struct PrefixMerge {
    uint32_t row;
    uint32_t own0, own_stride, n_own;
    uint32_t pre0, pre_stride, n_pre;
    uint32_t pad;
};

struct PrefixLaunch {
    PoolGeom pool;
    const float* q;
    float* out;
    int64_t q_row_stride, q_layer_stride;
    int64_t out_row_stride, out_layer_stride;
    const uint8_t* plan;
    uint32_t off_items, off_table, off_merges;
    float* part_o;   // [partial][n_lay][n_head][head_dim]: unnormalised outputs
    float* part_ml;  // [partial][n_lay][n_head][2]: running maximum (log2) and sum
    uint32_t n_items, n_merges;
    uint32_t layer0, n_lay;
    uint32_t group;  // G
    uint32_t wide;       // items of up to kWideSlots * waves slots of a prefix, else of up to kSlotTile
    uint32_t waves;      // wide: waves of slots; row_slots: waves of an item (2, 4)
    uint32_t row_slots;  // 1, 2: every item is one row of at most this many slots; 0: not so
    float qscale;    // log2(e) / sqrt(head_dim)
};
hipError_t launch_prefix_attention(const PrefixLaunch& a, const void* inline_plan, uint32_t inline_bytes,
                                   hipStream_t s, const LaunchTiming& t = {});
hipError_t launch_prefix_merge(const PrefixLaunch& a, const void* inline_plan, uint32_t inline_bytes, hipStream_t s,
                               const LaunchTiming& t = {});

// ------------------------------------------------------ draft verification

constexpr uint32_t kVerifyChunk = 2048;  // vocabulary entries one workgroup adds up

struct VerifyLaunch {
    const void* target;
    int64_t target_seq_stride, target_row_stride;
    const void* draft;  // null: the drafter names one token a step
    int64_t draft_seq_stride, draft_row_stride;
    const int32_t* drafted;
    int64_t drafted_stride;
    const int32_t* n_drafts;  // null: n_draft of every sequence
    const float* accept_u;
    int64_t accept_stride;
    const float* sample_u;
    int32_t* accepted;
    int32_t* tokens;
    int64_t tokens_stride;
    double* sums;  // [n_seq][chunks][2]: what is left of the target's row, and the row itself
    uint32_t n_seq, n_draft, vocab, dtype;
    uint32_t per;  // chunks one workgroup of the sums adds up
};
hipError_t launch_verify(const VerifyLaunch& a, hipStream_t s);

// ------------------------------------------------------------------ errors

// Set ni_kv_last_error(NULL) of this thread; returns `code`.
int call_error(int code, const char* fmt, ...) __attribute__((format(printf, 2, 3)));

}  // namespace ni
