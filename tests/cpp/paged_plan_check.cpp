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
    return find_row(x, t, *seq, *pos) ? 1 : 0;
}
int paged_sequence(const nvfp4_kv_cache* c, const nvfp4_paged_batch* b, int s, int* out) {
    Batch x{};
    if (int e = check_batch(c, b, &x)) return e;
    const Sequence q = sequence(x, s);
    out[0] = q.q0; out[1] = q.q_len; out[2] = q.first; out[3] = q.kv; out[4] = sees(q, 0); out[5] = sees(q, most(q.q_len - 1, 0));
    return 0;
}

// Walks the runs of all blocks over the batch's units.  0: runs are in order, none is empty, together they are all units; for every
// item the blocks that hold a part of it are those from block_of(first unit) to block_of(last unit), and each of them has a unit of it.
int paged_walk(const nvfp4_kv_cache* c, const nvfp4_paged_batch* b, int group, int chunk, int grid, int min_units) {
    Batch x{};
    if (check_batch(c, b, &x)) return 1;
    long long units = 0;
    std::vector<long long> begins;
    for (int s = 0; s < x.sequences; ++s) {
        const Items n = items_of(x, sequence(x, s), group, chunk, 0x7fffffff);
        for (int i = 0; i < n.items; ++i) begins.push_back(units + (long long)i * n.chunks);
        units += (long long)n.items * n.chunks;
    }
    begins.push_back(units);
    if (units == 0) return 0;
    const int blocks = blocks_of(units, grid, min_units);
    if (blocks < 1 || blocks > grid) return 2;
    for (int k = 0; k < blocks; ++k)
        if (run_begin(units, blocks, k) >= run_begin(units, blocks, k + 1)) return 3;
    if (run_begin(units, blocks, 0) != 0 || run_begin(units, blocks, blocks) != units) return 4;
    for (size_t i = 0; i + 1 < begins.size(); ++i) {
        const int first = block_of(units, blocks, begins[i]), last = block_of(units, blocks, begins[i + 1] - 1);
        if (first < 0 || last >= blocks || last < first) return 5;
        if (begins[i] < run_begin(units, blocks, first) || begins[i] >= run_begin(units, blocks, first + 1)) return 6;
        if (begins[i + 1] - 1 < run_begin(units, blocks, last) || begins[i + 1] - 1 >= run_begin(units, blocks, last + 1)) return 7;
    }
    return 0;
}

}  // extern "C"
