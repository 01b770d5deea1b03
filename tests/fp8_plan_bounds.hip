// Checks on the host that no plan of an 8-bit attention call leaves what the
// host provides for it: workgroups, partial entries, the workspace, the 31 bits
// of the device's sums (tests/test_fp8_plan_bounds.py).  It includes the
// library's host code, and the plan as the kernels take it from the sums over
// the requests.  Prints one line per check: its name and how many random calls
// broke it.
#include "../residualquant_amd/csrc/capi.hip"

#include <map>
#include <random>

namespace {

std::mt19937_64 g_rng(31);

int64_t below(int64_t n) { return (int64_t)(g_rng() % (uint64_t)n); }

// Log-uniform over low..high.
int64_t spread(double low, double high) {
    std::uniform_real_distribution<double> u(std::log(low), std::log(high + 1));
    return (int64_t)std::exp(u(g_rng));
}

std::map<std::string, int> g_broken;
void check(const char* name, bool holds) { g_broken[name] += holds ? 0 : 1; }

void call() {
    static const int kHeads[] = {1, 2, 3, 4, 8, 16, 16, 24, 55, 64, 128}, kGroups[] = {1, 1, 1, 2, 4, 7, 8, 16, 48};
    rq::Fp8AttentionParams p{};
    p.kv_heads = kHeads[below(11)];
    const int group = kGroups[below(9)];
    p.heads = p.kv_heads * group;
    p.head_dim = below(2) ? 128 : 96;
    p.page_tokens = below(2) ? 16 : 32;
    p.requests = below(10) ? spread(1, rq::kPlanRequests) : spread(65, 300);
    p.num_blocks = 1;
    const int64_t longest = below(20) ? spread(1, 60000) : spread(60000, 6000000);
    const int64_t shortest = spread(1, longest), most = below(4) ? spread(1, 1500) : 1;
    std::vector<int64_t> history, rows;
    for (int64_t b = 0; b < p.requests; ++b) {
        history.push_back(below(10) ? spread(shortest, longest) : 0);
        rows.push_back(below(3) ? most : below(most + 1));
        p.rows += rows.back();
    }
    if (p.rows == 0) p.rows = rows[0] = 1;
    p.rows += below(4) ? 0 : below(5);  // padding behind the last request
    p.max_pages = std::max<int64_t>(1, (longest + p.page_tokens - 1) / p.page_tokens + below(3) - 1);
    if (below(50) == 0) p.max_pages *= 1 + below(40);
    p.entries = fp8_entries(p.rows, p.heads, p.kv_heads, p.head_dim, p.max_pages, p.page_tokens);
    plan_fp8(p);
    const size_t bytes = rq_paged_attention_fp8_workspace_bytes(p.rows, p.heads, p.kv_heads, p.head_dim, p.max_pages, p.page_tokens);
    check("entries_in_workspace", 255 + sizeof(float) * (p.head_dim + 4) * p.kv_heads * (size_t)p.entries <= bytes);
    check("entries_in_32_bits", p.entries * (p.head_dim + 4) * 4 < (int64_t)1 << 31);
    // Columns, tiles and steps of the requests, as fp8_item takes them.
    std::vector<int64_t> columns, tiles, steps;
    int64_t total = 0, counts = 0, longest_steps = 0;
    for (int64_t b = 0; b < p.requests; ++b) {
        columns.push_back(rows[b] * group);
        tiles.push_back((columns[b] + p.tile - 1) / p.tile);
        steps.push_back((std::min(history[b], p.max_pages * p.page_tokens) + 31) / 32 + (rows[b] + 31) / 32);
        total += tiles[b] * steps[b];
        counts += tiles[b];
        if (tiles[b] > 0) longest_steps = std::max(longest_steps, steps[b]);
    }
    if (p.items == 0) {
        // Every slot of the grid takes `splits`; slot of request b: its first column / tile + b.
        const int64_t slots = p.rows * group / p.tile + p.requests;
        int64_t first = 0;
        for (int64_t b = 0; b < p.requests; ++b) {
            const int64_t slot = first / p.tile + b;
            check("slots", tiles[b] == 0 || slot + tiles[b] <= slots);
            check("slots_apart", tiles[b] == 0 || b + 1 == p.requests || slot + tiles[b] <= (first + columns[b]) / p.tile + b + 1);
            first += columns[b];
        }
        check("slot_entries", p.splits == 1 || p.rows * group * p.splits <= p.entries);
        return;
    }
    check("sums_in_31_bits", total < (int64_t)1 << 31);
    const rq::PlanSizes sizes = rq::fp8_sizes(p);
    const rq::PlanShare share = rq::plan_share_of(sizes, (uint32_t)total, (uint32_t)counts, (uint32_t)longest_steps);
    int64_t items = 0, entries = 0, most_splits = 1;
    for (int64_t b = 0; b < p.requests; ++b) {
        const int64_t splits = share.whole ? 1 : rq::plan_splits(sizes, share, (uint32_t)steps[b]);
        items += tiles[b] * splits;
        entries += columns[b] * splits;
        if (tiles[b] > 0) most_splits = std::max(most_splits, splits);
    }
    check("items", items <= p.items);
    // (The kernels write entries where a request is split; the number of an entry counts all requests.)
    check("entries", most_splits == 1 || entries <= p.entries);
    check("splits", most_splits <= std::max(p.plan_max_splits, p.splits) && most_splits <= kFp8MaxSplits);
    check("join_launched", most_splits == 1 || p.splits > 1 || p.plan_max_splits > 1);
}

}  // namespace

int main() {
    for (int i = 0; i < 200000; ++i) call();
    for (const auto& [name, broken] : g_broken) printf("%s %d\n", name.c_str(), broken);
}
