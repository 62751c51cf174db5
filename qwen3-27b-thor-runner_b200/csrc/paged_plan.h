// The batch over a paged cache: checks of the calls' arguments, where a position lies, and how the attention of few tokens shares its
// work among blocks.  Plain arithmetic, no CUDA types, so that a test can walk it on the CPU.
#pragma once
#include <cmath>
#include <cstdint>
#include <initializer_list>

#include "../../include/nvfp4_b200.h"

#ifdef __CUDACC__
#define NVFP4_PAGED_HD __host__ __device__ __forceinline__
#else
#define NVFP4_PAGED_HD inline
#endif

namespace nvfp4 {
namespace paged {

constexpr unsigned int kStatusPlace = 0xA01u;      // a page number or position out of bounds was left out
// What a handle reports: a wait that ran out, whose results are worth nothing, before a place that was left out.
inline unsigned int reported(unsigned int wait, unsigned int place) { return wait ? wait : place; }
constexpr int kMaxPositions = 0x7fffffff - 65536;  // positions are 32-bit numbers, with room for a tile behind the last one

template <class T>
NVFP4_PAGED_HD T least(T a, T b) { return a < b ? a : b; }
template <class T>
NVFP4_PAGED_HD T most(T a, T b) { return a < b ? b : a; }

// pos / page_size for 0 <= pos < 2^31 as a product and a shift: with l = ceil(log2 d) and mul = ceil(2^(31+l) / d) the quotient is
// exact, since the rounding of mul adds less than pos * 2^l / (d * 2^(31+l)) < 1 / d.
struct PageDivider {
    uint32_t mul;
    int shift;
};
inline PageDivider make_divider(int d) {
    int l = 0;
    while ((1LL << l) < d) ++l;
    return {(uint32_t)((((unsigned long long)1 << (31 + l)) + (unsigned)d - 1) / (unsigned)d), 31 + l};
}
NVFP4_PAGED_HD int divide(int pos, const PageDivider& p) { return (int)(((unsigned long long)(uint32_t)pos * p.mul) >> p.shift); }

// A cache and a batch after validation; strides in elements of two bytes.
struct Batch {
    const int *cu_q, *kv_len, *table;
    long long table_stride;
    int table_cols, sequences, tokens, max_q_len;
    uint16_t *k, *v;
    int num_pages, page_size, kv_heads, head_dim;
    long long page_stride, token_stride, head_stride;
    int max_kv;                        // table_cols * page_size
    PageDivider div;
    unsigned int* status;              // the handle's status word: the first wait that ran out
    unsigned int* places;              // and its word for places out of bounds, so that these hide no wait
};

struct Sequence {
    int q0, q_len;      // rows of the new tokens
    int first;          // position of the first of them (negative: padded)
    int kv;             // positions 0 .. kv - 1 may be read
};

NVFP4_PAGED_HD Sequence sequence(const Batch& b, int s) {
    int q0 = s, q1 = s + 1;
    if (b.cu_q) {
        q0 = b.cu_q[s];
        q1 = b.cu_q[s + 1];
    }
    Sequence r;
    r.q0 = least(most(q0, 0), b.tokens);
    r.q_len = least(most(q1, r.q0), b.tokens) - r.q0;
    const int kv = b.kv_len[s];
    // row r.q0 is row q0 unless cu_q was out of bounds
    const long long first = (long long)kv - ((long long)q1 - r.q0);
    r.first = (int)least(most(first, -2147483647LL), 2147483647LL);
    r.kv = least(most(kv, 0), b.max_kv);
    return r;
}

// Whether sequence() leaves something out: rows outside [0, tokens], or positions behind the table of a sequence that has rows.
NVFP4_PAGED_HD bool cut_off(const Batch& b, int s) {
    if (b.cu_q) {
        const int q0 = b.cu_q[s], q1 = b.cu_q[s + 1];
        if (q0 < 0 || q1 < q0 || q1 > b.tokens) return true;
        if (q0 == q1) return false;
    }
    return b.kv_len[s] > b.max_kv;
}

// The keys that new token i of a sequence sees are those in front of this position.
NVFP4_PAGED_HD int sees(const Sequence& q, int i) { return (int)most(least((long long)q.first + i + 1, (long long)q.kv), 0LL); }

// Element offset of the first value of a position (0 <= pos < max_kv) within k and v, head 0; -1 where its page is none.
NVFP4_PAGED_HD long long place(const Batch& b, int s, int pos) {
    const int entry = divide(pos, b.div);
    const int page = b.table[(long long)s * b.table_stride + entry];
    if ((unsigned)page >= (unsigned)b.num_pages) return -1;
    return (long long)page * b.page_stride + (long long)(pos - entry * b.page_size) * b.token_stride;
}

// The position of row t of sequence s, [q0, q1) its rows by cu_q; false where the row is none of the sequence's or its position is negative.
NVFP4_PAGED_HD bool row_position(const Batch& b, int s, int q0, int q1, int t, int& pos) {
    if (t < q0 || t >= q1) return false;
    const long long p = (long long)b.kv_len[s] - ((long long)q1 - t);
    pos = (int)p;
    return p >= 0;
}

// ---- work of the attention of few tokens.  An item is a (sequence, key-value head, tile of 16 rows); it takes `chunks` units of `chunk`
// tokens each.  All units in order (sequence, head, tile, chunk) are cut into equal runs, one per block.
constexpr int kRows = 16;
//
// What an item costs beside its units (its rows of q, the warps' sums, the result's way out) is about item_cost() units, so that a run of
// many short items would take several times as long as a run of a long one: runs are cut in places of cost, of which an item has
// item_cost() in front of its units.  A window of more than item_cost() places holds a unit, so no run is without one.  Measured: 64 sequences,
// heads of 256, cost 2, 3, 4: 88.8, 84.4, 83.8 us; one sequence of 1501 tokens 15.5, 16.6, 17.6; 243 sequences, heads of 128: 107, 109, 117.
NVFP4_PAGED_HD int item_cost(int head_dim) { return head_dim == 256 ? 3 : 2; }
struct Items {
    int tiles, items, chunks, extra;
    NVFP4_PAGED_HD int cost() const { return chunks + extra; }                  // of one item
};
NVFP4_PAGED_HD Items items_of(const Batch& b, const Sequence& q, int group, int chunk, int most_rows) {
    Items n{0, 0, 1, item_cost(b.head_dim)};
    const long long rows = (long long)q.q_len * group;
    if (rows > 0 && rows <= most_rows) {
        n.tiles = (int)((rows + kRows - 1) / kRows);
        n.items = n.tiles * b.kv_heads;
        n.chunks = most((q.kv + chunk - 1) / chunk, 1);
    }
    return n;
}
// Blocks in use: no more than there are runs of min_cost (more than an item costs beside its units) places.
NVFP4_PAGED_HD int blocks_of(long long cost, int grid, int min_cost) { return (int)least((long long)grid, most(cost / min_cost, 1LL)); }
NVFP4_PAGED_HD long long run_begin(long long cost, int blocks, int block) { return cost * block / blocks; }
// The block whose run holds place c.
NVFP4_PAGED_HD int block_of(long long cost, int blocks, long long c) { return (int)(((c + 1) * blocks - 1) / cost); }
// The units [from, to) of an item at place `at` that lie in the run [c0, c1).
struct Units {
    int from, to;
};
NVFP4_PAGED_HD Units units_in(long long at, const Items& n, long long c0, long long c1) {
    const long long u = at + n.extra;
    return {(int)least(most(c0 - u, 0LL), (long long)n.chunks), (int)least(most(c1 - u, 0LL), (long long)n.chunks)};
}
// An item that several blocks share is held in parts by blocks first .. first + count - 1: the first one's part, the only one of an item that
// begins in that block and is split, in its slot 1, the others' in their slots 0.
constexpr int kMaxBlocks = 256;
NVFP4_PAGED_HD int part_slot(int first, int block) { return 2 * block + (block == first ? 1 : 0); }

// ---- work of the attention of many tokens.  An item is a (sequence, tile of tile_tokens new tokens, key-value head); its units are the
// kLongChunk keys wide chunks that its last token sees, so a prompt's tiles have more and more of them.  Items in order (sequence, tile, head) have
// long_cost() places of cost in front of their units and are cut into runs as above.  Measured with a cost of 2, 4, 6: a prompt of 8192 tokens, heads of
// 256, 1098, 835, 804 us; a mixed step with heads of 128 107, 105, 112.
constexpr int kLongChunk = 128;
NVFP4_PAGED_HD int long_cost(int head_dim) { return head_dim == 256 ? 6 : 4; }

// sum of floor((a i + b) / m) over 0 <= i < n (m > 0, a (n - 1) + b and a mod m * n + b mod m below 2^32).  The published method for such sums: whole parts
// of slope and offset are summed at once, and the points below the line that is left are counted along the other axis, which swaps slope and modulus as in Euclid's
// algorithm (the reciprocity of floor sums, as in Graham, Knuth, Patashnik, Concrete Mathematics, 3.5)
NVFP4_PAGED_HD long long floor_sum(uint32_t n, uint32_t m, uint32_t a, uint32_t b) {
    long long sum = 0;
    while (n > 0) {
        sum += (long long)n * (n - 1) / 2 * (a / m) + (long long)n * (b / m);
        a %= m;
        b %= m;
        const uint32_t top = a * n + b;
        if (top < m) break;
        n = top / m;
        b = top % m;
        const uint32_t t = m;
        m = a;
        a = t;
    }
    return sum;
}

struct LongItems {
    int tiles, tile_tokens, heads, extra;
};
NVFP4_PAGED_HD LongItems long_items_of(const Batch& b, const Sequence& q, int group, int tile_tokens, int above_rows) {
    LongItems n{0, tile_tokens, b.kv_heads, long_cost(b.head_dim)};
    if ((long long)q.q_len * group > above_rows) n.tiles = (q.q_len + tile_tokens - 1) / tile_tokens;
    return n;
}
// Keys that the last token of a tile sees, and the tile's units (one at least: rows that see nothing have a result too).
NVFP4_PAGED_HD int long_limit(const Sequence& q, const LongItems& n, int tile) {
    return sees(q, (int)least((long long)(tile + 1) * n.tile_tokens, (long long)q.q_len) - 1);
}
NVFP4_PAGED_HD int long_chunks(int limit) { return most((limit + kLongChunk - 1) / kLongChunk, 1); }
// Places of the first `tiles` tiles of one head.
NVFP4_PAGED_HD long long long_places(const Sequence& q, const LongItems& n, int tiles) {
    const int full = least(tiles, n.tiles - 1), step = n.tile_tokens;             // tiles whose last token is (i + 1) * step - 1
    long long sum = (long long)tiles * n.extra;
    if (tiles == n.tiles && tiles > 0) sum += long_chunks(long_limit(q, n, tiles - 1));
    if (full <= 0) return sum;
    // first + (i + 1) * step keys: up to kLongChunk of them one chunk, beyond kv those that kv has
    const int ones = least((int)least(most((long long)kLongChunk - q.first, 0LL), 0x7fffffffLL) / step, full);
    const int open = least((int)least(most((long long)q.kv - q.first, 0LL), 0x7fffffffLL) / step, full);
    sum += ones;
    if (open > ones) sum += floor_sum((uint32_t)(open - ones), kLongChunk, (uint32_t)step, (uint32_t)(q.first + (ones + 1) * step + kLongChunk - 1));
    const int past = full - most(open, ones);
    return sum + (long long)past * long_chunks(q.kv);
}

// ---- checks of the calls' arguments
inline bool aligned(const void* p, unsigned n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

// The bytes from the first to behind the last value of a strided tensor.
struct Span {
    uintptr_t from = 0, to = 0;
    bool overlaps(const Span& o) const { return from && o.from && from < o.to && o.from < to; }
};
inline Span span_of(const void* p, long long rows, long long stride, long long heads, long long head_stride, int dim) {
    if (!p || rows <= 0 || heads <= 0) return {};
    const uintptr_t c = reinterpret_cast<uintptr_t>(p);
    return {c, c + (uintptr_t)((rows - 1) * stride + (heads - 1) * head_stride + dim) * 2};
}
// Indices lo .. hi of a stride.
struct Steps {
    long long stride, lo, hi;
};
inline long long floor_quotient(long long a, long long b) { return a / b - (a % b != 0 && a < 0); }
// Whether two runs of `dim` values whose distance is d and some index of each of n strides (above 0) have a value in common.  Exact: of the largest
// stride only the indices are tried that the others can still bring near, which is one or two where the strides are nested, as those of rows are.  A search
// of more than `budget` steps, which takes strides that no layout has, counts as found.
inline bool meet(long long d, const Steps* t, int n, int dim, int& budget) {
    if (--budget < 0) return true;
    if (n == 0) return d > -dim && d < dim;
    long long low = 0, high = 0;
    for (int i = 1; i < n; ++i) {
        low += t[i].stride * t[i].lo;
        high += t[i].stride * t[i].hi;
    }
    // -dim < d + i * stride + (low .. high) < dim
    const long long from = most(floor_quotient(-dim - d - high, t->stride) + 1, t->lo), to = least(-floor_quotient(d + low - dim, t->stride) - 1, t->hi);
    for (long long i = from; i <= to; ++i)
        if (meet(d + i * t->stride, t + 1, n - 1, dim, budget)) return true;
    return false;
}
inline bool meet(long long d, std::initializer_list<Steps> strides, int dim) {
    Steps t[4];
    int n = 0, budget = 1 << 16;
    for (const Steps& x : strides) {
        if (x.lo == 0 && x.hi == 0) continue;
        int i = n++;
        for (; i > 0 && t[i - 1].stride < x.stride; --i) t[i] = t[i - 1];
        t[i] = x;
    }
    return meet(d, t, n, dim, budget);
}
// Two tensors of `rows` rows whose spans overlap: whether they share a value.
inline bool rows_meet(const void* p, long long stride, long long heads, long long head_stride, const void* q, long long q_stride, long long q_heads, long long q_head_stride,
                      long long rows, int dim) {
    const long long d = (static_cast<const char*>(p) - static_cast<const char*>(q)) / 2;
    if (stride == q_stride) return meet(d, {{stride, 1 - rows, rows - 1}, {head_stride, 0, heads - 1}, {q_head_stride, 1 - q_heads, 0}}, dim);
    return meet(d, {{stride, 0, rows - 1}, {q_stride, 1 - rows, 0}, {head_stride, 0, heads - 1}, {q_head_stride, 1 - q_heads, 0}}, dim);
}
// Whether two places of a tensor that is written, any two indices of its strides, share a value.  (Strides nested in any order, the usual case, are
// told apart at once.)
inline bool repeats(std::initializer_list<Steps> strides, int dim) {
    Steps t[3];
    int n = 0;
    for (const Steps& x : strides) {                 // by rising stride
        if (x.hi <= 0) continue;
        int i = n++;
        for (; i > 0 && t[i - 1].stride > x.stride; --i) t[i] = t[i - 1];
        t[i] = x;
    }
    long long extent = dim;
    bool nested = true;
    for (int i = 0; i < n; ++i) {
        nested = nested && t[i].stride >= extent;
        extent += t[i].stride * t[i].hi;
    }
    if (nested) return false;
    // two indices differ first in stride i, there by one or more
    for (int i = 0; i < n; ++i) {
        Steps u[3] = {{1, 0, 0}, {1, 0, 0}, {1, 0, 0}};
        for (int j = i; j < n; ++j) u[j] = {t[j].stride, j == i ? 1 : -t[j].hi, t[j].hi};
        if (meet(0, {u[0], u[1], u[2]}, dim)) return true;
    }
    return false;
}
// n steps of a stride stay far from the end of 64 bits
inline bool fits(long long n, long long stride) { return n <= 0 || stride <= (1LL << 46) / n; }

// Stride defaults and rules of a [rows][heads][dim] tensor.
inline int check_strides(const void* p, long long& stride, long long& head_stride, long long rows, long long heads, int dim) {
    if (!head_stride) head_stride = dim;
    if (!stride) stride = heads * dim;
    if (stride < dim || head_stride < dim || !fits(rows, stride) || !fits(heads, head_stride)) return NVFP4_E_SHAPE;
    return !aligned(p, 16) || (stride & 7) || (head_stride & 7) ? NVFP4_E_ALIGN : NVFP4_OK;
}

inline int check_batch(const nvfp4_kv_cache* c, const nvfp4_paged_batch* b, Batch* out) {
    if (!c || !b) return NVFP4_E_NULL;
    if (b->sequences < 0 || b->tokens < 0 || b->max_q_len < 0) return NVFP4_E_SHAPE;
    if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256) return NVFP4_E_SHAPE;
    if (c->kv_heads < 1 || c->kv_heads > 65536 || c->page_size < 1 || c->num_pages < 1) return NVFP4_E_SHAPE;
    if (b->table_cols < 1 || (b->sequences > 1 && b->table_stride < b->table_cols) || !fits(b->sequences, b->table_stride)) return NVFP4_E_SHAPE;
    if ((long long)b->table_cols * c->page_size > kMaxPositions) return NVFP4_E_SHAPE;
    if (!b->cu_q && b->tokens < b->sequences) return NVFP4_E_SHAPE;
    // a stride that no index multiplies may be anything that is not negative
    if (c->page_stride < (c->num_pages > 1 ? c->head_dim : 0) || c->token_stride < (c->page_size > 1 ? c->head_dim : 0) ||
        c->head_stride < (c->kv_heads > 1 ? c->head_dim : 0))
        return NVFP4_E_SHAPE;
    if (!fits(c->num_pages, c->page_stride) || !fits(c->page_size, c->token_stride) || !fits(c->kv_heads, c->head_stride)) return NVFP4_E_SHAPE;
    if (b->tokens > 0 && b->sequences > 0) {
        if (!c->k || !c->v || !b->kv_len || !b->block_table) return NVFP4_E_NULL;
        if (!aligned(c->k, 16) || !aligned(c->v, 16) || ((c->page_stride | c->token_stride | c->head_stride) & 7)) return NVFP4_E_ALIGN;
        if (!aligned(b->cu_q, 4) || !aligned(b->kv_len, 4) || !aligned(b->block_table, 4)) return NVFP4_E_ALIGN;
    }
    *out = Batch{b->cu_q, b->kv_len, b->block_table, b->table_stride, b->table_cols, b->sequences, b->tokens, b->max_q_len,
                 static_cast<uint16_t*>(c->k), static_cast<uint16_t*>(c->v), c->num_pages, c->page_size, c->kv_heads, c->head_dim,
                 c->page_stride, c->token_stride, c->head_stride, b->table_cols * c->page_size, make_divider(c->page_size), nullptr, nullptr};
    return NVFP4_OK;
}
inline Span span_of_cache(const Batch& b, const void* p) {
    const uintptr_t c = reinterpret_cast<uintptr_t>(p);
    return {c, c + (uintptr_t)((b.num_pages - 1) * b.page_stride + (b.page_size - 1) * b.token_stride + (b.kv_heads - 1) * b.head_stride + b.head_dim) * 2};
}

// The calls' arguments after validation.
struct AppendArgs {
    Batch b;
    const uint16_t *q, *k, *v;
    uint16_t* q_out;
    long long q_stride, q_head, k_stride, k_head, v_stride, v_head, o_stride, o_head;
    const uint16_t *q_norm, *k_norm;
    const float* inv_freq;
    const int* positions;
    int q_heads, rot_dim;
    float eps;
};
struct AttentionArgs {
    Batch b;
    const uint16_t *q, *gate;
    uint16_t* out;
    long long q_stride, q_head, g_stride, g_head, o_stride, o_head;
    int q_heads, group;
    float scale;
};

// *empty: the call is right and has nothing to do.
inline int check_append(const nvfp4_kv_append_desc* d, AppendArgs* out, bool* empty) {
    if (!d) return NVFP4_E_NULL;
    AppendArgs a{};
    if (int e = check_batch(d->cache, d->batch, &a.b)) return e;
    const int dim = a.b.head_dim, tokens = a.b.tokens;
    if (d->q_heads < 0 || d->q_heads > 65536 || d->rot_dim < 0 || d->rot_dim > dim || (d->rot_dim & 15) != 0) return NVFP4_E_SHAPE;
    if ((d->q_norm || d->k_norm) && !(d->norm_eps >= 0.0f)) return NVFP4_E_SHAPE;
    *empty = tokens == 0 || a.b.sequences == 0;
    if (*empty) return NVFP4_OK;
    const bool has_q = d->q_heads > 0;
    if (!d->k || !d->v || (has_q && (!d->q || !d->q_out)) || (d->rot_dim && !d->inv_freq)) return NVFP4_E_NULL;
    a.q = has_q ? static_cast<const uint16_t*>(d->q) : nullptr;
    a.q_out = has_q ? static_cast<uint16_t*>(d->q_out) : nullptr;
    a.k = static_cast<const uint16_t*>(d->k);
    a.v = static_cast<const uint16_t*>(d->v);
    a.q_stride = d->q_stride; a.q_head = d->q_head_stride;
    a.k_stride = d->k_stride; a.k_head = d->k_head_stride;
    a.v_stride = d->v_stride; a.v_head = d->v_head_stride;
    a.o_stride = d->q_out_stride; a.o_head = d->q_out_head_stride;
    if (has_q) {
        if (int e = check_strides(a.q, a.q_stride, a.q_head, tokens, d->q_heads, dim)) return e;
        if (int e = check_strides(a.q_out, a.o_stride, a.o_head, tokens, d->q_heads, dim)) return e;
        if (repeats({{a.o_stride, 0, tokens - 1}, {a.o_head, 0, d->q_heads - 1}}, dim)) return NVFP4_E_SHAPE;
    }
    if (int e = check_strides(a.k, a.k_stride, a.k_head, tokens, a.b.kv_heads, dim)) return e;
    if (int e = check_strides(a.v, a.v_stride, a.v_head, tokens, a.b.kv_heads, dim)) return e;
    if (repeats({{a.b.page_stride, 0, a.b.num_pages - 1}, {a.b.token_stride, 0, a.b.page_size - 1}, {a.b.head_stride, 0, a.b.kv_heads - 1}}, dim)) return NVFP4_E_SHAPE;
    if (!aligned(d->q_norm, 16) || !aligned(d->k_norm, 16) || !aligned(d->inv_freq, 4) || !aligned(d->positions, 4)) return NVFP4_E_ALIGN;
    // in place: the same rows and heads, each read and written by the same thread
    const bool in_place = has_q && a.q == a.q_out && a.q_stride == a.o_stride && a.q_head == a.o_head;
    const Span q = span_of(a.q, tokens, a.q_stride, d->q_heads, a.q_head, dim), o = span_of(a.q_out, tokens, a.o_stride, d->q_heads, a.o_head, dim);
    const Span k = span_of(a.k, tokens, a.k_stride, a.b.kv_heads, a.k_head, dim), v = span_of(a.v, tokens, a.v_stride, a.b.kv_heads, a.v_head, dim);
    const Span ck = span_of_cache(a.b, a.b.k), cv = span_of_cache(a.b, a.b.v);
    // keys and values may lie between one another (pages that hold both), but not in one another
    if (ck.overlaps(cv) && meet(a.b.k - a.b.v, {{a.b.page_stride, 1 - a.b.num_pages, a.b.num_pages - 1}, {a.b.token_stride, 1 - a.b.page_size, a.b.page_size - 1},
                                                  {a.b.head_stride, 1 - a.b.kv_heads, a.b.kv_heads - 1}}, dim))
        return NVFP4_E_ALIAS;
    if (!in_place && (o.overlaps(q) || o.overlaps(k) || o.overlaps(v))) return NVFP4_E_ALIAS;
    // in place keys and values may lie between q's rows and heads, as a merged projection leaves them, but not in them
    if (in_place && o.overlaps(k) && rows_meet(a.q_out, a.o_stride, d->q_heads, a.o_head, a.k, a.k_stride, a.b.kv_heads, a.k_head, tokens, dim)) return NVFP4_E_ALIAS;
    if (in_place && o.overlaps(v) && rows_meet(a.q_out, a.o_stride, d->q_heads, a.o_head, a.v, a.v_stride, a.b.kv_heads, a.v_head, tokens, dim)) return NVFP4_E_ALIAS;
    for (const Span& x : {q, k, v, o})
        if (x.overlaps(ck) || x.overlaps(cv)) return NVFP4_E_ALIAS;
    a.q_norm = static_cast<const uint16_t*>(d->q_norm);
    a.k_norm = static_cast<const uint16_t*>(d->k_norm);
    a.inv_freq = d->inv_freq;
    a.positions = d->positions;
    a.q_heads = d->q_heads;
    a.rot_dim = d->rot_dim;
    a.eps = d->norm_eps;
    *out = a;
    return NVFP4_OK;
}

inline int check_attention(const nvfp4_paged_attention_desc* d, AttentionArgs* out, bool* empty) {
    if (!d) return NVFP4_E_NULL;
    AttentionArgs a{};
    if (int e = check_batch(d->cache, d->batch, &a.b)) return e;
    const int dim = a.b.head_dim, tokens = a.b.tokens;
    if (d->q_heads < 1 || d->q_heads > 65536 || d->q_heads % a.b.kv_heads != 0) return NVFP4_E_SHAPE;
    if (!std::isfinite(d->scale)) return NVFP4_E_SCALE;
    a.q_heads = d->q_heads;
    a.group = d->q_heads / a.b.kv_heads;
    if ((long long)tokens * a.group > kMaxPositions) return NVFP4_E_SHAPE;             // rows are 32-bit numbers
    *empty = tokens == 0 || a.b.sequences == 0;
    if (*empty) return NVFP4_OK;
    if (!d->q || !d->out) return NVFP4_E_NULL;
    a.q = static_cast<const uint16_t*>(d->q);
    a.gate = static_cast<const uint16_t*>(d->gate);
    a.out = static_cast<uint16_t*>(d->out);
    a.q_stride = d->q_stride; a.q_head = d->q_head_stride;
    a.g_stride = d->gate_stride; a.g_head = d->gate_head_stride;
    a.o_stride = d->out_stride; a.o_head = d->out_head_stride;
    if (int e = check_strides(a.q, a.q_stride, a.q_head, tokens, d->q_heads, dim)) return e;
    if (int e = check_strides(a.out, a.o_stride, a.o_head, tokens, d->q_heads, dim)) return e;
    if (repeats({{a.o_stride, 0, tokens - 1}, {a.o_head, 0, d->q_heads - 1}}, dim)) return NVFP4_E_SHAPE;
    if (a.gate)
        if (int e = check_strides(a.gate, a.g_stride, a.g_head, tokens, d->q_heads, dim)) return e;
    const Span o = span_of(a.out, tokens, a.o_stride, d->q_heads, a.o_head, dim);
    if (o.overlaps(span_of(a.q, tokens, a.q_stride, d->q_heads, a.q_head, dim)) || o.overlaps(span_of(a.gate, tokens, a.g_stride, d->q_heads, a.g_head, dim)) ||
        o.overlaps(span_of_cache(a.b, a.b.k)) || o.overlaps(span_of_cache(a.b, a.b.v)))
        return NVFP4_E_ALIAS;
    a.scale = d->scale != 0.0f ? d->scale : 1.0f / std::sqrt((float)dim);
    *out = a;
    return NVFP4_OK;
}

}  // namespace paged
}  // namespace nvfp4
