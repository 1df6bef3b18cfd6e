// Host-side checks of the operators on ragged new tokens over a paged cache,
// shared by the device and the GPU-free validation entry point.
#pragma once

#include "plan.h"

namespace slhip {

// Host copies of the u32 buffers that a call names.
struct PagedTables {
    const uint32_t* row_starts = nullptr;
    const uint32_t* seq_lens = nullptr;
    const uint32_t* block_table = nullptr;
};

// A call's arguments: `q`, `out` and `k`, `v` as the operator has them.
struct PagedCall {
    uint32_t kind = 0;  // sl_paged_kind
    const sl_op* op = nullptr;
    const sl_op* rope = nullptr;
    const sl_paged_tokens* tokens = nullptr;
    const sl_paged_kv* kv = nullptr;
    const sl_buffer_ref* q = nullptr;
    const sl_buffer_ref* k = nullptr;
    const sl_buffer_ref* v = nullptr;
    const sl_buffer_ref* out = nullptr;
    uint32_t window = 0, sinks = 0, prefix = 0;
};

// What the launch is sized for.
struct PagedPlan {
    // The most keys that one row's queries see, and the query rows per KV head (each row's counted
    // up to whole blocks), of the rows with up to `few` query rows and of the others; the others'
    // blocks of 256; rows with tokens.
    uint32_t few_keys = 0, many_keys = 0;
    uint64_t few_keys_in_all = 0, many_keys_in_all = 0;
    uint64_t few_rows = 0, many_rows = 0, many_blocks = 0, rows_with_tokens = 0;
};

// A pointer that the operator cannot do without is null.
bool paged_argument_missing(const PagedCall& c);
// Everything about the arguments, buffers and ranges; true when the tables'
// contents can be looked at.
bool check_paged_call(const BufferView& buffers, const PagedCall& c, Error* err);
// The contents of the row starts, lengths and block tables, after
// check_paged_call.
bool check_paged_contents(const PagedCall& c, const PagedTables& t, uint32_t few, PagedPlan* plan, Error* err);

}  // namespace slhip
