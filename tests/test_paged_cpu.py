"""The paged cache's calls as far as the CPU can check them: refusals, places and bounds, and the work lists of the attention of few tokens."""
import ctypes
import os
import random
import subprocess

import numpy as np
import pytest

import nvfp4

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
E_NULL, E_SHAPE, E_ALIGN, E_ALIAS, E_SCALE = -1, -2, -3, -5, -6
BASE = 1 << 20       # an address; nothing is read from it here


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    out = str(tmp_path_factory.mktemp("paged") / "paged_plan_check.so")
    subprocess.run(["g++", "-std=c++17", "-O2", "-Wall", "-Wextra", "-Werror", "-shared", "-fPIC", "-fsanitize=undefined", "-fno-sanitize-recover",
                    "-I", os.path.join(ROOT, "qwen3-27b-thor-runner_b200", "csrc"), "-o", out,
                    os.path.join(ROOT, "tests", "cpp", "paged_plan_check.cpp")], check=True)
    l = ctypes.CDLL(out)
    l.paged_wrong_quotients.restype = ctypes.c_longlong
    return l


def cache(**over):
    c = nvfp4.KvCacheStruct(BASE << 8, BASE << 9, 100, 16, 2, 128, 16 * 256, 256, 128)
    for k, v in over.items():
        setattr(c, k, v)
    return c


def batch(**over):
    b = nvfp4.PagedBatchStruct(BASE, BASE, BASE, 8, 8, 3, 40, 20)
    for k, v in over.items():
        setattr(b, k, v)
    return b


def append_desc(c=None, b=None, **over):
    c, b = c or cache(), b or batch()
    d = nvfp4.KvAppendDesc(ctypes.addressof(c), ctypes.addressof(b), BASE << 1, BASE << 2, BASE << 3, BASE << 4)
    d.q_heads, d.rot_dim, d.inv_freq, d.q_norm, d.k_norm, d.norm_eps = 8, 64, BASE, BASE, BASE, 1e-6
    for k, v in over.items():
        setattr(d, k, v)
    d.keep = (c, b)
    return d


def attention_desc(c=None, b=None, **over):
    c, b = c or cache(), b or batch()
    d = nvfp4.PagedAttentionDesc(ctypes.addressof(c), ctypes.addressof(b), BASE << 1, BASE << 2, BASE << 3)
    d.q_heads = 8
    for k, v in over.items():
        setattr(d, k, v)
    d.keep = (c, b)
    return d


def check(lib, d):
    empty = ctypes.c_int(-1)
    f = lib.paged_check_append if isinstance(d, nvfp4.KvAppendDesc) else lib.paged_check_attention
    return f(ctypes.byref(d), ctypes.byref(empty)), empty.value


SHARED_REFUSALS = [
    (dict(head_dim=96), {}, E_SHAPE), (dict(head_dim=0), {}, E_SHAPE), (dict(kv_heads=0), {}, E_SHAPE), (dict(page_size=0), {}, E_SHAPE),
    (dict(page_size=-16), {}, E_SHAPE), (dict(num_pages=0), {}, E_SHAPE), (dict(token_stride=64), {}, E_SHAPE), (dict(head_stride=0), {}, E_SHAPE),
    (dict(page_stride=0), {}, E_SHAPE), (dict(page_stride=-4096), {}, E_SHAPE), (dict(page_stride=1 << 45), {}, E_SHAPE),
    (dict(token_stride=260), {}, E_ALIGN), (dict(k=(BASE << 8) + 8), {}, E_ALIGN), (dict(v=(BASE << 9) + 2), {}, E_ALIGN), (dict(k=None), {}, E_NULL),
    (dict(v=None), {}, E_NULL),
    ({}, dict(sequences=-1), E_SHAPE), ({}, dict(tokens=-1), E_SHAPE), ({}, dict(max_q_len=-1), E_SHAPE), ({}, dict(table_cols=0), E_SHAPE),
    ({}, dict(table_stride=7), E_SHAPE), ({}, dict(table_cols=1 << 27, table_stride=1 << 27), E_SHAPE), ({}, dict(cu_q=None, tokens=2), E_SHAPE),
    ({}, dict(kv_len=None), E_NULL), ({}, dict(block_table=None), E_NULL), ({}, dict(kv_len=BASE + 2), E_ALIGN), ({}, dict(cu_q=BASE + 1), E_ALIGN),
    ({}, dict(block_table=BASE + 3), E_ALIGN),
]


@pytest.mark.parametrize("c,b,status", SHARED_REFUSALS)
def test_refusals_of_cache_and_batch(lib, c, b, status):
    assert check(lib, append_desc(cache(**c), batch(**b)))[0] == status
    assert check(lib, attention_desc(cache(**c), batch(**b)))[0] == status


@pytest.mark.parametrize("over,status", [
    (dict(cache=None), E_NULL), (dict(batch=None), E_NULL), (dict(k=None), E_NULL), (dict(v=None), E_NULL), (dict(q=None), E_NULL), (dict(q_out=None), E_NULL),
    (dict(inv_freq=None), E_NULL), (dict(q_heads=-1), E_SHAPE), (dict(rot_dim=24), E_SHAPE), (dict(rot_dim=144), E_SHAPE), (dict(rot_dim=-16), E_SHAPE),
    (dict(norm_eps=-1.0), E_SHAPE), (dict(norm_eps=float("nan")), E_SHAPE), (dict(q_stride=64), E_SHAPE), (dict(q_head_stride=64), E_SHAPE),
    (dict(k_stride=-256), E_SHAPE), (dict(v_stride=260), E_ALIGN), (dict(q_out_head_stride=132), E_ALIGN), (dict(q=(BASE << 1) + 8), E_ALIGN),
    (dict(q_norm=BASE + 8), E_ALIGN), (dict(k_norm=BASE + 2), E_ALIGN), (dict(inv_freq=BASE + 2), E_ALIGN), (dict(positions=BASE + 1), E_ALIGN),
    (dict(q_out=(BASE << 1) + 16), E_ALIAS), (dict(q_out=BASE << 2), E_ALIAS), (dict(q_out=BASE << 3), E_ALIAS), (dict(q_out=BASE << 8), E_ALIAS),
    (dict(q_out=(BASE << 9) + 4096), E_ALIAS), (dict(k=BASE << 8), E_ALIAS), (dict(q_out=BASE << 1, q_out_stride=1032), E_ALIAS),
])
def test_append_refusals(lib, over, status):
    assert check(lib, append_desc(**over))[0] == status


@pytest.mark.parametrize("over,status", [
    (dict(cache=None), E_NULL), (dict(batch=None), E_NULL), (dict(q=None), E_NULL), (dict(out=None), E_NULL), (dict(q_heads=0), E_SHAPE), (dict(q_heads=7), E_SHAPE),
    (dict(scale=float("inf")), E_SCALE), (dict(scale=float("nan")), E_SCALE), (dict(q_stride=512), 0), (dict(q_stride=64), E_SHAPE), (dict(out_stride=-1024), E_SHAPE),
    (dict(gate=(BASE << 2) + 8), E_ALIGN), (dict(gate_head_stride=132), E_ALIGN), (dict(out=BASE << 1), E_ALIAS), (dict(out=(BASE << 2) + 64), E_ALIAS),
    (dict(out=BASE << 8), E_ALIAS), (dict(out=BASE << 9), E_ALIAS), (dict(q_stride=1 << 44), E_SHAPE),
])
def test_attention_refusals(lib, over, status):
    assert check(lib, attention_desc(**over))[0] == status


def test_calls_that_are_right(lib):
    assert check(lib, append_desc()) == (0, 0) and check(lib, attention_desc()) == (0, 0)
    assert check(lib, append_desc(q_out=BASE << 1)) == (0, 0)                                   # in place
    assert check(lib, append_desc(q=None, q_out=None, q_heads=0)) == (0, 0)                     # keys and values only
    assert check(lib, append_desc(rot_dim=0, inv_freq=None, q_norm=None, k_norm=None, norm_eps=-1.0)) == (0, 0)
    assert check(lib, attention_desc(gate=None)) == (0, 0)
    for b in (batch(tokens=0), batch(sequences=0)):
        b.kv_len = b.block_table = None
        c = cache(k=None, v=None)
        assert check(lib, append_desc(c, b, k=None)) == (0, 1) and check(lib, attention_desc(c, b, q=None)) == (0, 1)
    # strides that nothing is multiplied with
    assert check(lib, attention_desc(cache(kv_heads=1, head_stride=0), q_heads=8)) == (0, 0)
    assert check(lib, attention_desc(cache(page_size=1, token_stride=0))) == (0, 0)


def test_entry_points_refuse_a_missing_handle():
    lib = nvfp4.load()
    assert lib.nvfp4_kv_append(None, None, None) == -1 and lib.nvfp4_paged_attention(None, None, None) == -1


def test_descriptor_layouts(tmp_path):
    """The binding's structures have the header's sizes and offsets."""
    src = tmp_path / "layout.c"
    pairs = [("nvfp4_kv_cache", nvfp4.KvCacheStruct), ("nvfp4_paged_batch", nvfp4.PagedBatchStruct), ("nvfp4_kv_append_desc", nvfp4.KvAppendDesc),
             ("nvfp4_paged_attention_desc", nvfp4.PagedAttentionDesc)]
    lines = [f"_Static_assert(sizeof({n}) == {ctypes.sizeof(s)}, \"size\");" for n, s in pairs]
    lines += [f"_Static_assert(offsetof({n}, {f[0]}) == {getattr(s, f[0]).offset}, \"{n}.{f[0]}\");" for n, s in pairs for f in s._fields_]
    src.write_text('#include "nvfp4_b200.h"\n' + "\n".join(lines) + "\n")
    subprocess.run(["gcc", "-std=c11", "-c", "-o", str(tmp_path / "layout.o"), "-I", os.path.join(ROOT, "include"), str(src)], check=True)


@pytest.mark.parametrize("d", [1, 2, 3, 5, 7, 16, 24, 40, 48, 63, 64, 65, 127, 1000, 65537, (1 << 30) + 1, 0x7fffffff])
def test_page_quotients(lib, d):
    assert lib.paged_wrong_quotients(d, 300000) == 0


def arrays(kv, table, cu=None, tokens=None, **c):
    kv, table = np.asarray(kv, np.int32), np.ascontiguousarray(table, np.int32)
    cu = None if cu is None else np.asarray(cu, np.int32)
    b = nvfp4.PagedBatchStruct(None if cu is None else cu.ctypes.data, kv.ctypes.data, table.ctypes.data, table.shape[1], table.shape[1], len(kv),
                               len(kv) if tokens is None else tokens, 1)
    b.keep = (kv, table, cu)
    return cache(**c), b


def test_bad_pages_have_no_place(lib):
    """Page numbers out of bounds, at both ends and beyond 32 bits' sign, and lengths behind the table."""
    c, b = arrays([30, 9, 100], [[0, 1, 2], [-1, 0, 0], [9, 10, -2147483648]], num_pages=10, page_size=8, page_stride=8 * 256)
    out = (ctypes.c_longlong * 100)()
    assert lib.paged_places(ctypes.byref(c), ctypes.byref(b), 0, 40, out) == 24              # clamped to three pages
    assert [out[i] for i in range(24)] == [p // 8 * 2048 + p % 8 * 256 for p in range(24)] and out[24] == -2
    assert lib.paged_places(ctypes.byref(c), ctypes.byref(b), 1, 9, out) == 9
    assert [out[i] for i in range(9)] == [-1] * 8 + [0]
    assert lib.paged_places(ctypes.byref(c), ctypes.byref(b), 2, 24, out) == 24
    assert [out[i] for i in range(24)] == [9 * 2048 + i * 256 for i in range(8)] + [-1] * 16
    # far offsets: the product is formed in 64 bits
    c, b = arrays([5], [[0x7ffffffe]], num_pages=0x7fffffff, page_size=8, page_stride=1 << 14)
    assert lib.paged_places(ctypes.byref(c), ctypes.byref(b), 0, 5, out) == 5 and out[4] == (0x7ffffffe << 14) + 4 * 256


def test_rows_and_sequences(lib):
    seq, pos = ctypes.c_int(), ctypes.c_int()
    cu = [2, 2, 7, 7, 8, 12]
    c, b = arrays([0, 9, 4, 0, 4], [[0]] * 5, cu=cu, tokens=15, page_size=64)
    got = []
    for t in range(15):
        ok = lib.paged_row(ctypes.byref(c), ctypes.byref(b), t, ctypes.byref(seq), ctypes.byref(pos))
        got.append((seq.value, pos.value) if ok else None)
    # two rows in front, sequence 1 at 4..8, sequence 3 of length 0 has no position, sequence 4 at 0..3, three padded rows
    assert got == [None, None] + [(1, 4 + i) for i in range(5)] + [None] + [(4, i) for i in range(4)] + [None] * 3
    out = (ctypes.c_int * 6)()
    for s, want in enumerate([(2, 0, 0, 0), (2, 5, 4, 9), (7, 0, 4, 4), (7, 1, -1, 0), (8, 4, 0, 4)]):
        assert lib.paged_sequence(ctypes.byref(c), ctypes.byref(b), s, out) == 0 and tuple(out[:4]) == want
    assert lib.paged_sequence(ctypes.byref(c), ctypes.byref(b), 1, out) == 0 and tuple(out[4:]) == (5, 9)
    assert lib.paged_sequence(ctypes.byref(c), ctypes.byref(b), 3, out) == 0 and tuple(out[4:]) == (0, 0)


def test_offsets_out_of_bounds_are_clamped(lib):
    out = (ctypes.c_int * 6)()
    rng = random.Random(3)
    wild = [-2147483648, -5, 0, 3, 9, 10, 11, 500, 2147483647]
    for _ in range(500):
        cu, kv = [rng.choice(wild) for _ in range(4)], [rng.choice(wild) for _ in range(3)]
        c, b = arrays(kv, [[0, 1]] * 3, cu=cu, tokens=10, page_size=16)
        for s in range(3):
            assert lib.paged_sequence(ctypes.byref(c), ctypes.byref(b), s, out) == 0
            q0, n, _, k, lo, hi = out
            assert 0 <= q0 and 0 <= n and q0 + n <= 10 and 0 <= k <= 32 and 0 <= lo <= k and 0 <= hi <= k
        seq, pos = ctypes.c_int(), ctypes.c_int()
        for t in range(10):
            if lib.paged_row(ctypes.byref(c), ctypes.byref(b), t, ctypes.byref(seq), ctypes.byref(pos)):
                assert 0 <= seq.value < 3 and pos.value >= 0 and cu[seq.value] <= t < cu[seq.value + 1]


def test_every_unit_has_one_block(lib):
    rng = random.Random(11)
    for _ in range(400):
        n = rng.choice([1, 2, 5, 40, 300])
        new = [rng.choice([0, 1, 1, 1, 2, 5, 30]) for _ in range(n)]
        kv = [rng.choice([0, x, x + rng.randint(0, 300), x + rng.randint(0, 5000)]) for x in new]
        c, b = arrays(kv, np.zeros((n, 400), np.int32), cu=np.cumsum([0] + new), tokens=sum(new) + 1, page_size=16, kv_heads=rng.choice([1, 2, 8]))
        got = lib.paged_walk(ctypes.byref(c), ctypes.byref(b), rng.choice([1, 3, 12, 16]), rng.choice([64, 128]), rng.choice([1, 2, 148, 256]), rng.choice([4, 9]))
        assert got == 0, (got, new, kv)


def test_places_of_causal_tiles(lib):
    """The closed form of the units of a prompt's tiles: behind a past, at its own start, with rows in front of position 0, cut off by the page table."""
    rng = random.Random(12)
    for _ in range(3000):
        q = rng.choice([1, 2, 127, 128, 129, rng.randint(1, 300), rng.randint(1, 9000)])
        kv = rng.choice([0, q, q + rng.randint(0, 300), q + rng.randint(0, 200000), rng.randint(0, q), -5, 2147483647])
        max_kv = rng.choice([2147418111, rng.randint(1, 400), rng.randint(1, 20000)])
        step = rng.choice([1, 2, 10, 21, 32, 128, 256, rng.randint(1, 256)])
        assert lib.paged_long_places(q, kv, max_kv, step) == 0, (q, kv, max_kv, step)


def test_the_binding_refuses_tensors_that_do_not_fit():
    """What the pointers cannot tell the library.  No call reaches it."""
    torch = pytest.importorskip("torch")
    h = object.__new__(nvfp4.Handle)                    # without a device: every call below ends in front of the library
    h.h, h.lib = None, None
    new = lambda *s, dtype=torch.bfloat16: torch.zeros(s, dtype=dtype)
    k = new(4, 16, 2, 64)
    cache = nvfp4.KvCache(k, k.clone())
    kv, table = torch.ones(3, dtype=torch.int32), torch.zeros(3, 2, dtype=torch.int32)
    batch = nvfp4.PagedBatch(kv, table)
    q, kn = new(3, 6, 64), new(3, 2, 64)
    for args in [(q, new(3, 1, 64), kn, q.clone()), (q, kn, new(3, 4, 64), q.clone()), (q, kn, new(3, 2, 32), q.clone()), (q, new(2, 2, 64), kn, q.clone()), (q, kn, kn, new(3, 4, 64)),
                 (new(3, 6, 32), kn, kn, new(3, 6, 32)), (new(2, 6, 64), kn, kn, q), (q, kn, new(1, 2, 64).expand(3, 2, 64), q.clone()),
                 (q, kn, new(3, 2, 128)[..., ::2], q.clone())]:
        with pytest.raises(ValueError):
            h.kv_append(cache, batch, *args)
    for args, kw in [((q, new(3, 4, 64)), {}), ((q, new(2, 6, 64)), {}), ((q, q.clone()), {"gate": new(3, 5, 64)}), ((new(3, 6, 32), new(3, 6, 32)), {}), ((new(3, 6, 128), new(3, 6, 128)), {}),
                     ((q, q.clone()), {"gate": new(3, 6, 32)})]:
        with pytest.raises(ValueError):
            h.paged_attention(cache, batch, *args, **kw)
    for bad in [lambda: nvfp4.KvCache(k, new(4, 16, 2, 128)), lambda: nvfp4.KvCache(k.float(), k.float()), lambda: nvfp4.KvCache(k, k, order="page"),
                lambda: nvfp4.KvCache(k[..., ::2], k[..., ::2]), lambda: nvfp4.PagedBatch(kv.long(), table), lambda: nvfp4.PagedBatch(kv, table[:2]),
                lambda: nvfp4.PagedBatch(kv, table, cu_q=kv), lambda: nvfp4.PagedBatch(kv.float(), table)]:
        with pytest.raises(ValueError):
            bad()
