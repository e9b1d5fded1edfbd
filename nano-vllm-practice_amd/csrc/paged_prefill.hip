// Chunked / varlen / causal paged prefill attention and dense flash
// attention: planning and launches of the tile kernel in attention_tiles.h.
#include "attention_tiles.h"

namespace femto {

static int pick_group(int n_rep) { return (n_rep % 4 == 0) ? 4 : (n_rep % 2 == 0) ? 2 : 1; }

// Query tiles per (kv head, head group) are at most num_tokens / BT plus one
// partial tile per sequence.
static int prefill_items_per_group(int num_seqs, int num_tokens, int BT) { return (num_tokens + BT - 1) / BT + num_seqs; }

hipError_t prefill_resident_workgroups(int& resident) {
    // Two workgroups per CU are resident (LDS and register budget).
    int cus = 0;
    const hipError_t e = device_cu_count(cus);
    if (e != hipSuccess) return e;
    resident = 2 * cus;
    return hipSuccess;
}

// A split call has at most `resident` pieces in all: one counter and one
// partial slot per resident workgroup, whatever the batch.  (As many counters
// again for the decode rows' merge: a call that needs more takes the merge
// launch.)
size_t prefill_counter_bytes(int resident) { return ((size_t)resident * 2 * sizeof(int) + 255) & ~(size_t)255; }

size_t prefill_workspace_bytes(int resident) {
    return resident > 0 ? prefill_counter_bytes(resident) + (size_t)resident * kPartSlotBytes : 0;
}

int prefill_group(int n_rep) { return pick_group(n_rep); }

hipError_t launch_paged_prefill(int dtype, PrefillArgs a, int num_tokens, int decode_rows_max, hipStream_t st) {
    const int G = pick_group(a.n_rep);
    const int BT = 32 * (4 / G);
    a.head_groups = a.n_rep / G;
    a.items_per_group = prefill_items_per_group(a.num_seqs, num_tokens, BT);
    a.tiles_per_group = a.items_per_group;
    a.total_work = a.tiles_per_group * a.n_kv_heads * a.head_groups;
    if (num_tokens <= 0 || a.num_seqs <= 0) return hipSuccess;
    {
        hipError_t e = prefill_resident_workgroups(a.resident);
        if (e != hipSuccess) return e;
    }
    if (a.decode_blocks > 0 && !a.skip_decode_rows) return hipErrorInvalidValue;
    const bool rows = a.window > 0 || a.fp4;  // what a.decode_blocks run
    if (a.decode_blocks > 0 && !rows && a.dec.head_groups * G != a.n_rep) return hipErrorInvalidValue;
    a.decode_blocks = (a.decode_blocks + 7) / 8 * 8;
    // Rows under the window in the same launch: the tiles are cut for one slot
    // of every CU, and rows run in the other from the start, half a slot's worth
    // of them ahead of the tiles (rows_first), the rest behind them; rows load
    // while tiles compute.  Rows seeing 1028 keys (32 query heads on 8) beside
    // 1024 new tokens behind 4096, us: 127 rows 131 with tiles cut for both
    // slots and ahead of all rows, 114 with all rows ahead of them, 100 so; 33
    // rows 68, 57 and 46; 4 rows 43, 38 and 38.  Every second or third
    // workgroup a row: 100-125.  Over 192 shapes (16-200 rows, 512-4000 new tokens,
    // windows of 1024 and 4096, 64/8, 32/8 and 16/8 heads) all rows ahead is 4 %
    // slower at the median and up to 53 % (64 rows seeing 4100 keys beside 1024
    // tokens 157 and 242).  It is 0-7 % faster where the tiles about fill whole rounds of
    // both slots (2000 tokens beside 127 rows 136 and 129), 20-38 % slower where they
    // are a few more (1100 beside 64 rows of 16/8 heads 52 and 72): the host, which
    // knows a lower bound of their number only, cannot tell these apart.
    const int slots = a.resident;
    // Over a 4-bit cache a row is short against a chunk's tiles, and as many rows as
    // CUs run ahead of them (32/8 heads, 1024 tokens behind 4096 beside 127 rows of
    // 512-8192 keys: 162 us, all first 205, none 168).  Where the rows or
    // the tiles do not fill the CUs, the tiles stay cut for both slots, behind
    // all rows: beside 4 rows 81 and 97, beside 31 92 and 107; 512 tokens beside 127
    // 109 and 123.  Over 100 such shapes this is 3 % at the mean from the best of
    // nine orders; the host's one view of long and short rows costs most (16/8 heads,
    // 2048 behind 8192: beside 31 rows 151, with one slot 189, but beside 127 210
    // with 128 first and 215).
    const int tile_tokens = a.skip_decode_rows ? std::max(0, num_tokens - decode_rows_max) : num_tokens;
    const int64_t min_tiles = (int64_t)((tile_tokens + BT - 1) / BT) * a.n_kv_heads * a.head_groups;
    const bool both_slots = a.fp4 && (2 * a.decode_blocks <= slots || 2 * min_tiles < slots);
    if (rows && a.decode_blocks > 0 && !both_slots) a.resident /= 2;
    if (a.part) {
        // A split needs all pieces in the resident slots at once, and a call
        // has at least ceil(num_tokens / BT) query tiles per KV head group
        // (not counting sequences of one token when the decode workers take
        // them): when those already fill the slots the call cannot split, and
        // the kernel skips its split estimate.
        if (min_tiles >= a.resident) {
            a.part = nullptr;
            a.counters = nullptr;
        } else {
            // a split call has at most `resident` pieces
            a.total_work = a.total_work > a.resident ? a.total_work : a.resident;
        }
    }
    if (rows) {
        const int first = both_slots ? a.decode_blocks : a.fp4 ? slots / 2 : slots / 4;
        a.rows_first = std::min(a.decode_blocks, first) / 8 * 8;
        return a.fp4 ? launch_fp4_tiles(dtype, G, a, st) : launch_window_tiles(dtype, G, a, st);
    }
    hipError_t e = launch_dtype<true, kAllPages>(dtype, G, a, st);
    if (e == hipSuccess && a.decode_blocks > 0 && !a.dec.merge_counters) e = launch_paged_decode_merge(dtype, a.dec, a.num_seqs, st);
    return e;
}

hipError_t launch_dense_attention(int dtype, PrefillArgs a, hipStream_t st) {
    const int G = pick_group(a.n_rep);
    const int BT = 32 * (4 / G);
    a.head_groups = a.n_rep / G;
    a.tiles_per_group = a.num_seqs * ((a.q_len + BT - 1) / BT);
    a.total_work = a.tiles_per_group * a.n_kv_heads * a.head_groups;
    if (a.q_len <= 0 || a.num_seqs <= 0) return hipSuccess;
    return launch_dtype<false, kAllPages>(dtype, G, a, st);
}

}  // namespace femto
