// The plan of a batch's cross attention, on the host: from the lengths of its graphs,
// which workgroup takes which rows and keys.
#include <algorithm>
#include <cstring>
#include <string>
#include <vector>

#include "attention.h"
#include "internal.h"

namespace relm_mp {

namespace {

// Workgroups of a launch at least, where the lengths allow: four to each of 256 CUs, two of
// those that keep 64 or more rows (keys: 128) in registers.  Measured, us: one query over
// 2,000,000 keys, 8 / 2 heads of 64 in half precision, 270 at 256, 186 at 512, 208 at 1024, 200 at 2048
// (262,147 keys: 38, 29, 37, 34: 512 would serve these two better); large ones, 4 x 2048 x 4096
// with 4 heads of 128 in bfloat16, 153 at 256, 102 at 512, 113 at 1024, in training with heads of 64
// 313, 228, 259.
constexpr int64_t kWorkgroups = 1024;
constexpr int64_t kLargeWorkgroups = 512;
constexpr int64_t kPartUnit = 128;     // parts end on whole tiles of keys and rows
// Of a part: shorter ones cost more to join than to walk.  The query above over 32,000 keys: 11.9 us at
// 128, 11.1 at 256, 13.8 at 512, 17.3 at 1024 (over 2000: 10.6, 10.9, 11.8, 16.4).
constexpr int64_t kLeastKeys = 512;
// The same for rows: 5003 queries over 40 keys in training take 70 to 71 us at 128 to 1024 and 142 at 4096.
constexpr int64_t kLeastRows = 256;
constexpr int64_t kIdleKeys = 1024;    // of an item of a graph without queries, whose keys get zeros: at most 1 MB of them

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

int64_t padded(const std::vector<int64_t>& n, int64_t tile) {
    int64_t sum = 0;
    for (int64_t v : n) sum += ceil_div(v, tile) * tile;
    return sum;
}

struct Layout {
    std::vector<AttnItem> items, idle, key_items;
    std::vector<AttnJoin> joins, key_joins;
    int32_t row_tile = 16, key_tile = 64;
    int32_t num_parts = 0, num_key_parts = 0;
};

// Units [0, n) of one item in equal parts of about `share`, each but the last a
// multiple of kPartUnit: the number of parts and the units of one.
struct Split {
    int64_t parts, size;
};
Split split(int64_t n, int64_t share) {
    if (2 * n < 3 * share) return {1, n};
    const int64_t size = ceil_div(ceil_div(n, ceil_div(n, share)), kPartUnit) * kPartUnit;
    return {ceil_div(n, size), size};
}

// The order of items of unequal length: each XCD runs through an eighth of the list
// (work_of), so the items are dealt to eight parts of about the same total, and each part
// starts with its longest, so that none starts when the others end.  Items of one length
// stay in their graphs' order: neighbours read the same keys.
template <typename F>
void deal(std::vector<AttnItem>& items, F&& length) {
    const auto longer = [&](const AttnItem& a, const AttnItem& b) { return length(a) > length(b); };
    if (items.empty()) return;
    const auto [least, most] = std::minmax_element(items.begin(), items.end(),
                                                   [&](const AttnItem& a, const AttnItem& b) { return length(a) < length(b); });
    if (length(*least) == length(*most)) return;
    std::stable_sort(items.begin(), items.end(), longer);
    constexpr size_t kParts = 8;
    std::vector<AttnItem> dealt;
    dealt.reserve(items.size());
    for (size_t part = 0; part < kParts; ++part)
        for (size_t round = 0; round * kParts < items.size(); ++round) {  // there and back
            const size_t i = round * kParts + (round % 2 == 0 ? part : kParts - 1 - part);
            if (i < items.size()) dealt.push_back(items[i]);
        }
    items.swap(dealt);
}

int lay_out(const int64_t* qo, const int64_t* ko, int64_t graphs, int64_t group, int64_t kv_heads, Layout& L) {
    std::vector<int64_t> rows(graphs), keys(graphs);
    int64_t most_rows = 0;
    for (int64_t b = 0; b < graphs; ++b) {
        rows[b] = (qo[b + 1] - qo[b]) * group;
        keys[b] = ko[b + 1] - ko[b];
        most_rows = std::max(most_rows, rows[b]);
        if (rows[b] > RELM_MP_MAX_ROWS)
            return set_error(RELM_MP_ERR_INVALID_ARGUMENT, "relm_mp attention plan: a graph has too many queries");
    }
    // Rows of an item.  Up to 32, its waves take different keys and a row's sums meet at
    // the end; from there on each wave has rows of its own, 16 or 32.  128 rows read a
    // key tile half as often as 64, unless the lengths leave a fifth more rows empty.
    // Measured, us (this tile and the next larger one): 512 graphs of up to 16 x 200, 2 heads of 64, 14.9
    // and 17.6 in bfloat16, 30 and 53 in float, in training 47 and 50, 121 and 144; up to 32 x 300, 4 heads
    // of 64, 37 and 32, 151 and 116, in training 131 and 155, 481 and 543.  64 and 128 rows of 8 heads of 64
    // over 1000 keys, bfloat16: of 65 rows 41 and 37, of 150 33 and 37, of 1000 25 and 30; float: 175 and
    // 157, 125 and 152, 89 and 88; 4 x 2048 rows over 4096 keys, 16 / 4 heads of 128 in bfloat16, 437 and 338.
    // Keys, in training: of 150 70 and 73 in bfloat16, 267 and 313 in float.  (One graph of more than 32
    // rows moves a whole batch: 2048 graphs of up to 32, 33 and 64 rows take 290, 353 and 360 us in training.)
    if (most_rows <= 16)
        L.row_tile = 16;
    else if (most_rows <= 32)
        L.row_tile = 32;
    else
        L.row_tile = 5 * padded(rows, 128) <= 6 * padded(rows, 64) ? 128 : 64;
    L.key_tile = 5 * padded(keys, 128) <= 6 * padded(keys, 64) ? 128 : 64;

    // A share is what a workgroup gets when all the work is dealt to them.
    using Work = unsigned __int128;  // rows, keys and heads of 2^31, 2^31 and 2^12
    Work row_work = 0, key_work = 0;
    for (int64_t b = 0; b < graphs; ++b) {
        row_work += static_cast<Work>(ceil_div(rows[b], L.row_tile)) * keys[b] * kv_heads;
        key_work += static_cast<Work>(ceil_div(keys[b], L.key_tile)) * rows[b] * kv_heads;
    }
    const auto share = [](Work work, int64_t workgroups, int64_t least) {
        const Work s = (work + workgroups - 1) / workgroups;
        return s > RELM_MP_MAX_ROWS ? int64_t{RELM_MP_MAX_ROWS} : std::max(least, static_cast<int64_t>(s));
    };
    const int64_t key_share = share(row_work, L.row_tile >= 64 ? kLargeWorkgroups : kWorkgroups, kLeastKeys);
    const int64_t row_share = share(key_work, L.key_tile == 128 ? kLargeWorkgroups : kWorkgroups, kLeastRows);

    // table records: 512 MB of them at most, counted before any is made
    constexpr int64_t kMost = int64_t{1} << 24;
    int64_t records = 0;
    for (int64_t b = 0; b < graphs; ++b) {
        const int64_t row_parts = split(keys[b], key_share).parts, key_parts = split(rows[b], row_share).parts;
        records += ceil_div(rows[b], L.row_tile) * (row_parts + (row_parts > 1 ? 1 : 0));
        records += ceil_div(keys[b], L.key_tile) * (key_parts + (key_parts > 1 ? 1 : 0));
        if (rows[b] == 0) records += ceil_div(keys[b], kIdleKeys);
        if (records > kMost)
            return set_error(RELM_MP_ERR_INVALID_ARGUMENT, "relm_mp attention plan: too many queries and keys for one plan");
    }
    for (int64_t b = 0; b < graphs; ++b) {
        const Split s = split(keys[b], key_share);
        for (int64_t r = 0; r < rows[b]; r += L.row_tile) {
            const int32_t n = static_cast<int32_t>(std::min<int64_t>(L.row_tile, rows[b] - r));
            if (s.parts > 1)
                L.joins.push_back({static_cast<int32_t>(qo[b]), static_cast<int32_t>(r), n, 0, 0, L.num_parts,
                                   static_cast<int32_t>(s.parts), 0});
            for (int64_t p = 0; p < s.parts; ++p)
                L.items.push_back({static_cast<int32_t>(qo[b]), static_cast<int32_t>(r), n,
                                   static_cast<int32_t>(ko[b] + p * s.size),
                                   static_cast<int32_t>(std::min(s.size, keys[b] - p * s.size)),
                                   s.parts > 1 ? L.num_parts++ : -1, {}});
        }
        for (int64_t k = 0; rows[b] == 0 && k < keys[b]; k += kIdleKeys)
            L.idle.push_back({static_cast<int32_t>(qo[b]), 0, 0, static_cast<int32_t>(ko[b] + k),
                              static_cast<int32_t>(std::min(kIdleKeys, keys[b] - k)), -1, {}});
        const Split t = split(rows[b], row_share);
        for (int64_t k = 0; k < keys[b]; k += L.key_tile) {
            const int32_t n = static_cast<int32_t>(std::min<int64_t>(L.key_tile, keys[b] - k));
            if (t.parts > 1)
                L.key_joins.push_back({static_cast<int32_t>(qo[b]), 0, 0, static_cast<int32_t>(ko[b] + k), n,
                                       L.num_key_parts, static_cast<int32_t>(t.parts), 0});
            for (int64_t p = 0; p < t.parts; ++p)
                L.key_items.push_back({static_cast<int32_t>(qo[b]), static_cast<int32_t>(p * t.size),
                                       static_cast<int32_t>(std::min(t.size, rows[b] - p * t.size)),
                                       static_cast<int32_t>(ko[b] + k), n, t.parts > 1 ? L.num_key_parts++ : -1, {}});
        }
    }
    deal(L.items, [](const AttnItem& i) { return i.keys; });
    // graphs of few rows have their backward in one kernel over the row items, but for float
    // rows of more than 64 values
    if (L.row_tile > 32) deal(L.key_items, [](const AttnItem& i) { return i.rows; });
    return RELM_MP_OK;
}

int check_offsets(const int64_t* o, int64_t graphs, int64_t rows, const char* name) {
    const auto bad = [&](const char* what) {
        return set_error(RELM_MP_ERR_INVALID_ARGUMENT, std::string("relm_mp attention plan: ") + name + what);
    };
    if (o[0] != 0 || o[graphs] != rows) return bad(" must run from 0 to the number of rows.");
    for (int64_t b = 0; b < graphs; ++b)
        if (o[b + 1] < o[b]) return bad(" must ascend.");
    return RELM_MP_OK;
}

}  // namespace

int build_attention_plan(const int64_t* qo, const int64_t* ko, int64_t graphs, int64_t q_rows, int64_t k_rows, int32_t heads,
                         int32_t kv_heads, void* table, size_t table_bytes, relm_mp_attention_plan* plan) {
    const auto bad = [](const char* what) {
        return set_error(RELM_MP_ERR_INVALID_ARGUMENT, std::string("relm_mp attention plan: ") + what);
    };
    if (plan == nullptr || graphs < 0 || (qo == nullptr) || (ko == nullptr)) return bad("NULL or negative argument");
    if (heads < 1 || kv_heads < 1 || heads > 4096 || heads % kv_heads != 0)
        return bad("heads must be a multiple of kv_heads, both in [1, 4096]");
    if (q_rows < 0 || k_rows < 0 || q_rows > RELM_MP_MAX_ROWS || k_rows > RELM_MP_MAX_ROWS)
        return bad("rows must be in [0, 2^31 - 2]");
    int rc = check_offsets(qo, graphs, q_rows, "q_offsets");
    if (rc == RELM_MP_OK) rc = check_offsets(ko, graphs, k_rows, "k_offsets");
    if (rc != RELM_MP_OK) return rc;
    Layout L;
    rc = lay_out(qo, ko, graphs, heads / kv_heads, kv_heads, L);
    if (rc != RELM_MP_OK) return rc;
    const size_t records = L.items.size() + L.idle.size() + L.joins.size() + L.key_items.size() + L.key_joins.size();
    relm_mp_attention_plan p{};
    p.q_rows = q_rows;
    p.k_rows = k_rows;
    p.heads = heads;
    p.kv_heads = kv_heads;
    p.graphs = graphs;
    p.table_bytes = static_cast<int64_t>(records * sizeof(AttnItem));
    p.row_tile = L.row_tile;
    p.key_tile = L.key_tile;
    p.num_items = static_cast<int32_t>(L.items.size());
    p.num_parts = L.num_parts;
    p.num_joins = static_cast<int32_t>(L.joins.size());
    p.num_key_items = static_cast<int32_t>(L.key_items.size());
    p.num_key_parts = L.num_key_parts;
    p.num_key_joins = static_cast<int32_t>(L.key_joins.size());
    p.num_idle_items = static_cast<int32_t>(L.idle.size());
    // a launch has fewer than 2^32 threads
    constexpr int64_t kMostBlocks = (int64_t{1} << 24) - 1;
    if (static_cast<int64_t>(std::max(L.items.size() + L.idle.size(), 2 * L.key_items.size())) * kv_heads > kMostBlocks ||
        static_cast<int64_t>(std::max(L.joins.size(), L.key_joins.size())) * 128 * kv_heads > kMostBlocks)
        return bad("too many items for one launch");
    *plan = p;
    if (table != nullptr) {
        if (table_bytes < static_cast<size_t>(p.table_bytes))
            return set_error(RELM_MP_ERR_WORKSPACE, "relm_mp attention plan: table too small");
        char* at = static_cast<char*>(table);
        const auto put = [&](const void* from, size_t n) {
            if (n > 0) std::memcpy(at, from, n * sizeof(AttnItem));
            at += n * sizeof(AttnItem);
        };
        put(L.items.data(), L.items.size());
        put(L.idle.data(), L.idle.size());
        put(L.joins.data(), L.joins.size());
        put(L.key_items.data(), L.key_items.size());
        put(L.key_joins.data(), L.key_joins.size());
    }
    return RELM_MP_OK;
}

}  // namespace relm_mp
