// What the attention kernels and the plan that lays their work out share.
#pragma once

#include <cstddef>
#include <cstdint>

#include "relm_mp.h"

namespace relm_mp {

// Rows of a graph: its queries times the heads that share a key head, row r being
// query r / group and head r % group of the key head.  A row item is a range of a
// graph's rows against a range of its keys, a key item a range of keys against a
// range of rows; every item is run once per key head.
struct AttnItem {
    int32_t q_first;    // the graph's first query
    int32_t row0;       // first row of the item within the graph
    int32_t rows;
    int32_t key_first;  // first key of the item in the batch
    int32_t keys;
    int32_t part;       // -1: the item's rows (keys) are whole; else where its sums go
    int32_t pad[2];
};

// Rows (keys) whose parts [part0, part0 + parts) are joined.
struct AttnJoin {
    int32_t q_first;
    int32_t row0;
    int32_t rows;
    int32_t key_first;
    int32_t keys;
    int32_t part0;
    int32_t parts;
    int32_t pad;
};
static_assert(sizeof(AttnItem) == 32 && sizeof(AttnJoin) == 32, "table records");

// The tables of a plan, one after the other; behind the row items the ranges of keys of
// graphs that have no queries.
inline const AttnItem* plan_items(const relm_mp_attention_plan& p) { return static_cast<const AttnItem*>(p.table); }
inline const AttnJoin* plan_joins(const relm_mp_attention_plan& p) {
    return reinterpret_cast<const AttnJoin*>(plan_items(p) + p.num_items + p.num_idle_items);
}
inline const AttnItem* plan_key_items(const relm_mp_attention_plan& p) {
    return reinterpret_cast<const AttnItem*>(plan_joins(p) + p.num_joins);
}
inline const AttnJoin* plan_key_joins(const relm_mp_attention_plan& p) {
    return reinterpret_cast<const AttnJoin*>(plan_key_items(p) + p.num_key_items);
}

// Where the parts' sums go: per part, key head and row (key) of its tile one row of
// head_dim floats, padded to 16 bytes (dk and dv: two); the forward's maxima and totals
// follow all rows.
inline int64_t attention_part_stride(int64_t head_dim) { return (head_dim + 3) / 4 * 4; }
inline int64_t attention_part_rows(const relm_mp_attention_plan& p) {
    return static_cast<int64_t>(p.num_parts) * p.kv_heads * p.row_tile;
}
inline size_t attention_part_floats(const relm_mp_attention_plan& p, int64_t head_dim) {
    return static_cast<size_t>(attention_part_rows(p) * (attention_part_stride(head_dim) + 2));
}
inline size_t attention_key_part_floats(const relm_mp_attention_plan& p, int64_t head_dim) {
    return static_cast<size_t>(p.num_key_parts) * p.kv_heads * p.key_tile * 2 * attention_part_stride(head_dim);
}

// What the forward keeps of a row for the backward: its largest score (not scaled) and one over
// the total of exp(scale * (s - top)).
struct RowStats {
    float top, inv_total;
};
static_assert(sizeof(RowStats) == 8, "two floats to a row");

struct AttnOperands {
    relm_mp_head_rows q, k, v, grad;
    int64_t head_dim;
    const uint8_t* key_mask;
    float scale;
    void* out;       // forward's output; the backward reads it
    float* lse;      // forward
    RowStats* stats;
    float* delta;    // backward: [q_rows, heads]
    void *dq, *dk, *dv;
    float* parts;
};

}  // namespace relm_mp
