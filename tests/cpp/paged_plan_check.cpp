// The paged cache's checks, places and work lists (csrc/paged_plan.h) for a test on the CPU.
#include <vector>

#include "paged_plan.h"

using namespace nvfp4::paged;

extern "C" {

int paged_check_append(const nvfp4_kv_append_desc* d, int* empty) {
    AppendArgs a{};
    bool e = false;
    const int st = check_append(d, &a, &e);
    *empty = e;
    return st;
}
int paged_check_attention(const nvfp4_paged_attention_desc* d, int* empty) {
    AttentionArgs a{};
    bool e = false;
    const int st = check_attention(d, &a, &e);
    *empty = e;
    return st;
}

// Positions 0 .. n - 1 and some near the end of the range whose quotient is not pos / d.
long long paged_wrong_quotients(int d, int n) {
    const PageDivider p = make_divider(d);
    long long bad = 0;
    for (int i = 0; i < n; ++i) bad += divide(i, p) != i / d;
    for (int i = 0; i < n; ++i) {
        const int pos = 0x7fffffff - i;
        bad += divide(pos, p) != pos / d;
        const int edge = (int)((long long)(0x7fffffff / d) * d - (i & 3));
        bad += edge >= 0 && divide(edge, p) != edge / d;
    }
    return bad;
}

// Element offset of every position of a sequence; the batch may hold anything (device memory in earnest).
int paged_places(const nvfp4_kv_cache* c, const nvfp4_paged_batch* b, int s, int n, long long* out) {
    Batch x{};
    if (int e = check_batch(c, b, &x)) return e;
    const Sequence q = sequence(x, s);
    for (int i = 0; i < n; ++i) out[i] = i < q.kv ? place(x, s, i) : -2;
    return q.kv;
}
int paged_row(const nvfp4_kv_cache* c, const nvfp4_paged_batch* b, int t, int* seq, int* pos) {
    Batch x{};
    if (int e = check_batch(c, b, &x)) return e;
    if (!x.cu_q) {
        *seq = t;
        return t < x.sequences && row_position(x, t, t, t + 1, t, *pos);
    }
    for (*seq = x.sequences - 1; *seq > 0 && x.cu_q[*seq] > t; --*seq) {}         // the last s with cu_q[s] <= t
    return row_position(x, *seq, x.cu_q[*seq], x.cu_q[*seq + 1], t, *pos);
}
int paged_sequence(const nvfp4_kv_cache* c, const nvfp4_paged_batch* b, int s, int* out) {
    Batch x{};
    if (int e = check_batch(c, b, &x)) return e;
    const Sequence q = sequence(x, s);
    out[0] = q.q0; out[1] = q.q_len; out[2] = q.first; out[3] = q.kv; out[4] = sees(q, 0); out[5] = sees(q, most(q.q_len - 1, 0));
    return 0;
}

// Places of a sequence's first tiles in closed form against the sum over them: the number of tiles at which the two differ.
int paged_long_places(int q_len, int kv_len, int max_kv, int tile_tokens) {
    Batch x{};
    x.tokens = q_len;
    x.kv_heads = 1;
    x.sequences = 1;
    x.max_kv = max_kv;
    const int cu[2] = {0, q_len};
    x.cu_q = cu;
    x.kv_len = &kv_len;
    const Sequence q = sequence(x, 0);
    const LongItems n = long_items_of(x, q, 1, tile_tokens, 0);
    long long sum = 0;
    int bad = long_places(q, n, 0) != 0;
    for (int t = 0; t < n.tiles; ++t) {
        const int limit = long_limit(q, n, t);
        if (limit < 0 || limit > q.kv) return -1;
        sum += long_chunks(limit) + long_cost(x.head_dim);
        bad += long_places(q, n, t + 1) != sum;
    }
    return bad;
}

// Walks the runs of all blocks over the batch's places of cost.  0: runs are in order and together all places, each holds a unit; the units of every
// item are shared among the blocks from that of its first unit to that of its last one, each of which has at least one, each unit once; no two
// parts of split items share a slot.
int paged_walk(const nvfp4_kv_cache* c, const nvfp4_paged_batch* b, int group, int chunk, int grid, int min_cost) {
    Batch x{};
    if (check_batch(c, b, &x)) return 1;
    long long cost = 0;
    std::vector<long long> at;
    std::vector<Items> items;
    for (int s = 0; s < x.sequences; ++s) {
        const Items n = items_of(x, sequence(x, s), group, chunk, 0x7fffffff);
        for (int i = 0; i < n.items; ++i) {
            at.push_back(cost + (long long)i * n.cost());
            items.push_back(n);
        }
        cost += (long long)n.items * n.cost();
    }
    if (cost == 0) return 0;
    const int blocks = blocks_of(cost, grid, min_cost);
    if (blocks < 1 || blocks > grid) return 2;
    if (run_begin(cost, blocks, 0) != 0 || run_begin(cost, blocks, blocks) != cost) return 3;
    std::vector<int> held(blocks, 0), slots(2 * blocks, 0);
    for (size_t i = 0; i < at.size(); ++i) {
        const Items& n = items[i];
        const int first = block_of(cost, blocks, at[i] + n.extra), last = block_of(cost, blocks, at[i] + n.extra + n.chunks - 1);
        if (first < 0 || last >= blocks || last < first) return 4;
        int next = 0;
        for (int k = first > 0 ? first - 1 : 0; k <= last + 1 && k < blocks; ++k) {
            const Units u = units_in(at[i], n, run_begin(cost, blocks, k), run_begin(cost, blocks, k + 1));
            if ((u.from < u.to) != (k >= first && k <= last)) return 5;
            if (u.from >= u.to) continue;
            if (u.from != next) return 6;
            next = u.to;
            ++held[k];
            if (last > first && ++slots[part_slot(first, k)] > 1) return 7;
        }
        if (next != n.chunks) return 8;
    }
    for (int k = 0; k < blocks; ++k)
        if (!held[k]) return 9;
    return 0;
}

}  // extern "C"
