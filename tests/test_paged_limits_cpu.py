"""The paged cache's calls at the ends of what they take, as far as the CPU can check them."""
import ctypes
import os
import random
import subprocess

import pytest
import torch

import nvfp4
import test_paged_cpu as base

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    out = str(tmp_path_factory.mktemp("paged") / "paged_limits_check.so")
    subprocess.run(["g++", "-std=c++17", "-O2", "-Wall", "-Wextra", "-Werror", "-shared", "-fPIC", "-fsanitize=undefined", "-fno-sanitize-recover",
                    "-I", os.path.join(ROOT, "qwen3-27b-thor-runner_b200", "csrc"), "-o", out,
                    os.path.join(ROOT, "tests", "cpp", "paged_limits_check.cpp")], check=True)
    return ctypes.CDLL(out)


def test_what_is_cut_off_is_noticed(lib):
    """Rows outside [0, tokens] and lengths behind the table, by the definition: for 10 rows and a table of 32 positions."""
    rng = random.Random(5)
    wild = [-2147483648, -5, 0, 3, 9, 10, 11, 500, 2147483647]
    seen = [0, 0]
    for _ in range(2000):
        cu, kv = sorted(rng.choice(wild) for _ in range(4)), [rng.choice(wild + [31, 32, 33]) for _ in range(3)]
        if rng.random() < 0.2:
            rng.shuffle(cu)
        c, b = base.arrays(kv, [[0, 1]] * 3, cu=cu, tokens=10, page_size=16)
        for s in range(3):
            rows_out = cu[s] < 0 or cu[s + 1] > 10 or cu[s + 1] < cu[s]
            want = rows_out or (cu[s + 1] > cu[s] and kv[s] > 32)
            assert lib.paged_cut_off(ctypes.byref(c), ctypes.byref(b), s) == want, (cu, kv, s)
            seen[want] += 1
    assert min(seen) > 200
    c, b = base.arrays([32, 33, 0, -1], [[0, 1]] * 4, page_size=16)            # a token a sequence
    assert [lib.paged_cut_off(ctypes.byref(c), ctypes.byref(b), s) for s in range(4)] == [0, 1, 0, 0]


class _Library:
    """Stands in for the library: keeps the descriptors that reach it."""

    def __init__(self):
        self.got = []

    def nvfp4_kv_append(self, handle, d, stream):
        self.got.append(nvfp4.KvAppendDesc.from_buffer_copy(d))
        return 0

    def nvfp4_paged_attention(self, handle, d, stream):
        self.got.append(nvfp4.PagedAttentionDesc.from_buffer_copy(d))
        return 0


def _bound(tokens=3, dim=64):
    """A handle on the stand-in, a cache and a batch of CPU tensors, and a function that makes zeros."""
    h = object.__new__(nvfp4.Handle)
    h.h, h.lib, h.device = None, _Library(), -1          # the device that CPU tensors name
    new = lambda *s, dtype=torch.bfloat16: torch.zeros(s, dtype=dtype)
    k = new(4, 16, 2, dim)
    batch = nvfp4.PagedBatch(torch.ones(tokens, dtype=torch.int32), torch.zeros(tokens, 2, dtype=torch.int32))
    return h, nvfp4.KvCache(k, k.clone()), batch, new


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.int16, torch.float64])
def test_the_binding_refuses_other_types_of_rows(dtype):
    h, cache, batch, new = _bound()
    with pytest.raises(ValueError):
        nvfp4.KvCache(new(4, 16, 2, 64, dtype=dtype), new(4, 16, 2, 64, dtype=dtype))
    rows = [new(3, 6, 64), new(3, 2, 64), new(3, 2, 64), new(3, 6, 64)]
    for i in range(4):
        bad = list(rows)
        bad[i] = bad[i].to(dtype)
        with pytest.raises(ValueError):
            h.kv_append(cache, batch, *bad, stream=0)
    q, out, gate = rows[0], rows[3], new(3, 6, 64)
    for args, kw in [((q.to(dtype), out), {}), ((q, out.to(dtype)), {}), ((q, out), {"gate": gate.to(dtype)})]:
        with pytest.raises(ValueError):
            h.paged_attention(cache, batch, *args, stream=0, **kw)
    assert not h.lib.got


def test_the_binding_refuses_vectors_that_do_not_fit():
    """Norms, frequencies and positions are read by the device without a look at what they are."""
    h, cache, batch, new = _bound()
    q, k, v, out = new(3, 6, 64), new(3, 2, 64), new(3, 2, 64), new(3, 6, 64)
    good = {"q_norm": new(64), "k_norm": new(64), "inv_freq": torch.ones(16), "positions": torch.arange(3, dtype=torch.int32)}
    h.kv_append(cache, batch, q, k, v, out, stream=0, **good)
    h.kv_append(cache, batch, q, k, v, out, stream=0)
    h.kv_append(cache, batch, None, k, v, None, stream=0, positions=torch.arange(9, dtype=torch.int32))
    assert [(d.q_norm, d.k_norm, d.inv_freq, d.positions) for d in h.lib.got[:2]] == [tuple(t.data_ptr() for t in good.values()), (None,) * 4]
    assert [(d.q_heads, d.rot_dim) for d in h.lib.got] == [(6, 32), (6, 0), (0, 0)]
    reached = len(h.lib.got)
    for name in ("q_norm", "k_norm"):
        for bad in [new(64, dtype=torch.float32), new(64, dtype=torch.float16), new(63), new(128), new(128)[::2], new(0)]:
            with pytest.raises(ValueError):
                h.kv_append(cache, batch, q, k, v, out, stream=0, **{**good, name: bad})
    for bad in [torch.ones(16, dtype=torch.float64), torch.ones(32)[::2], new(16)]:
        with pytest.raises(ValueError):
            h.kv_append(cache, batch, q, k, v, out, stream=0, **{**good, "inv_freq": bad})
    for bad in [torch.arange(3), torch.arange(2, dtype=torch.int32), torch.arange(6, dtype=torch.int32)[::2], torch.ones(3), torch.arange(3, dtype=torch.int16)]:
        with pytest.raises(ValueError):
            h.kv_append(cache, batch, q, k, v, out, stream=0, **{**good, "positions": bad})
    with pytest.raises(ValueError):
        h.kv_append(cache, batch, q, k, v, None, stream=0)
    kv, table = torch.ones(3, dtype=torch.int32), torch.zeros(3, 2, dtype=torch.int32)
    for args in [(kv.view(3, 1), table), (kv, torch.zeros(3, dtype=torch.int32)), (kv.to(torch.uint32), table), (kv, table.to(torch.uint32))]:
        with pytest.raises((ValueError, IndexError)):
            nvfp4.PagedBatch(*args)
    assert len(h.lib.got) == reached


def test_offsets_come_with_the_number_of_rows():
    """One row per sequence, the default without offsets, would leave out most of a prompt without a word."""
    kv, table, cu = torch.full((3,), 40, dtype=torch.int32), torch.zeros(3, 4, dtype=torch.int32), torch.tensor([0, 20, 21, 30], dtype=torch.int32)
    with pytest.raises(ValueError):
        nvfp4.PagedBatch(kv, table, cu_q=cu, max_q_len=20)
    assert nvfp4.PagedBatch(kv, table, tokens=30, cu_q=cu, max_q_len=20).tokens == 30
    assert nvfp4.PagedBatch(kv, table).tokens == 3 and nvfp4.PagedBatch(kv, table, tokens=5).tokens == 5


def test_the_binding_refuses_tensors_of_other_devices():
    """An address of the host's memory, or of another device's, would be read by the handle's device."""
    h, cache, batch, new = _bound()
    rows = [new(3, 6, 64), new(3, 2, 64), new(3, 2, 64), new(3, 6, 64)]
    h.kv_append(cache, batch, *rows, stream=0)
    h.paged_attention(cache, batch, rows[0], rows[3], stream=0)
    assert len(h.lib.got) == 2
    for on in [(0, -1, -1), (-1, 0, -1), (-1, -1, 0), (0, 0, -1), (0, 0, 0)]:           # of the handle, the cache and the batch; rows stay on the CPU
        h.device, cache.device, batch.device = on
        with pytest.raises(ValueError):
            h.kv_append(cache, batch, *rows, stream=0)
        with pytest.raises(ValueError):
            h.paged_attention(cache, batch, rows[0], rows[3], stream=0)
    assert len(h.lib.got) == 2
    h.device = cache.device = batch.device = -1
    for vector in ({"q_norm": new(64)}, {"inv_freq": torch.ones(16)}, {"positions": torch.arange(3, dtype=torch.int32)}):
        h.kv_append(cache, batch, *rows, stream=0, **vector)
        with pytest.raises(ValueError):
            h.kv_append(cache, batch, *rows, stream=0, **{n: _Elsewhere(t) for n, t in vector.items()})


class _Elsewhere:
    """A tensor that says it is on device 3."""

    def __init__(self, t):
        self.t = t

    def __getattr__(self, name):
        return getattr(self.t, name)

    def get_device(self):
        return 3


def test_the_current_stream_is_that_of_the_handles_device(monkeypatch):
    """The calls run on the handle's device, whichever is current; so does the stream that they take where none is given."""
    h, cache, batch, new = _bound()
    asked = []
    monkeypatch.setattr(nvfp4, "_raw_stream", lambda *device: asked.append(device) or 7)
    rows = [new(3, 6, 64), new(3, 2, 64), new(3, 2, 64), new(3, 6, 64)]
    h.kv_append(cache, batch, *rows)
    h.paged_attention(cache, batch, rows[0], rows[3])
    assert asked == [(-1,), (-1,)]
    assert nvfp4._stream(None) == 7 and asked[2] == (None,) and nvfp4._stream(5) == 5


def _values(at, rows, stride, heads, head_stride, dim):
    """The value numbers of a [rows][heads][dim] tensor."""
    return [at + r * stride + h * head_stride + i for r in range(rows) for h in range(heads) for i in range(dim)]


def test_keys_and_values_in_the_rows_of_queries_in_place(lib):
    """In place, keys and values may lie between q's rows and heads but not in them: against the sets of all values' places."""
    rng = random.Random(8)
    at, found = 1 << 22, [0, 0]
    for _ in range(1500):
        dim, rows, heads, kv_heads = 64, rng.choice([1, 2, 3, 5, 9]), rng.choice([1, 2, 3, 6]), rng.choice([1, 2, 3])
        heads = heads * kv_heads
        head = rng.choice([64, 64, 128, 136, 192])
        stride = rng.choice([(heads - 1) * head + 64, heads * head + kv_heads * 128, heads * head + 8 * rng.randint(0, 200)])
        k_head = rng.choice([64, 64, 72, 128, head, head])
        k_stride = rng.choice([stride, stride, stride, stride + 8, 2 * stride, 64 * kv_heads, k_head * kv_heads])
        k_at = 8 * rng.randint(-40, (rows * stride + heads * head) // 8 + 40)
        c = base.cache(k=1 << 30, v=1 << 31, head_dim=dim, kv_heads=kv_heads, head_stride=64, token_stride=64 * kv_heads, page_stride=16 * 64 * kv_heads)
        b = base.batch(tokens=rows)
        q = _values(0, rows, stride, heads, head, dim)
        want = not set(q).isdisjoint(_values(k_at, rows, k_stride, kv_heads, k_head, dim))
        for name, other in (("k", "v"), ("v", "k")):
            d = base.append_desc(c, b, q=at, q_out=at, q_heads=heads, rot_dim=0, q_stride=stride, q_head_stride=head, q_out_stride=stride, q_out_head_stride=head,
                                 **{name: at + 2 * k_at, name + "_stride": k_stride, name + "_head_stride": k_head, other: 1 << 26, other + "_stride": 64 * kv_heads})
            assert lib.limits_check_append(ctypes.byref(d)) == (base.E_ALIAS if want else 0), (rows, heads, head, stride, kv_heads, k_head, k_stride, k_at)
        found[want] += 1
    assert min(found) > 200
    # as a merged projection leaves them, 8192 tokens: q and gate head by head, then keys, then values
    c, b = base.cache(head_dim=256, head_stride=256, token_stride=512, page_stride=8192, k=1 << 40, v=1 << 41), base.batch(tokens=8192)
    row = (48 + 4) * 256
    good = dict(q=at, q_out=at, q_heads=24, rot_dim=0, q_stride=row, q_out_stride=row, q_head_stride=512, q_out_head_stride=512, k=at + 2 * 48 * 256, k_stride=row,
                v=at + 2 * 50 * 256, v_stride=row)
    assert lib.limits_check_append(ctypes.byref(base.append_desc(c, b, **good))) == 0
    for name, to in (("k", 47 * 256 - 8), ("v", 0), ("k", 256 * 46), ("v", 48 * 256 - 257 + 1), ("k", 49 * 256)):
        inside = not set(_values(0, 3, row, 24, 512, 256)).isdisjoint(_values(to, 3, row, 2, 256, 256))          # rows repeat: three tell
        status = lib.limits_check_append(ctypes.byref(base.append_desc(c, b, **{**good, name: at + 2 * to})))
        assert status == (base.E_ALIAS if inside else 0), (name, to)


def test_written_strides_that_repeat_a_place_are_refused(lib):
    """Two heads or tokens in one place would be written by two threads: q_out, out and the cache of the append against the sets of their values' places."""
    rng, dim, found = random.Random(9), 64, {"rows": [0, 0], "cache": [0, 0]}
    steps = [64, 64, 72, 96, 128, 136, 192, 256, 320, 384, 512, 640, 1024]
    for _ in range(2500):
        rows, heads = rng.choice([1, 2, 3, 4, 7]), rng.choice([1, 2, 3, 5, 8])
        stride, head = rng.choice(steps), rng.choice(steps)
        places = _values(0, rows, stride, heads, head, dim)
        want = base.E_SHAPE if len(set(places)) < len(places) else 0
        c, b = base.cache(kv_heads=1, head_dim=dim, token_stride=64, page_stride=1024), base.batch(tokens=rows)
        d = base.attention_desc(c, b, q_heads=heads, out_stride=stride, out_head_stride=head)
        assert lib.limits_check_attention(ctypes.byref(d)) == want, (rows, heads, stride, head)
        d = base.append_desc(c, b, q_heads=heads, rot_dim=0, q_out_stride=stride, q_out_head_stride=head)
        assert lib.limits_check_append(ctypes.byref(d)) == want, (rows, heads, stride, head)
        found["rows"][want != 0] += 1
        # what is read may repeat: a cache with heads in common is attended to, not appended to
        pages, page, kv_heads = rng.choice([1, 2, 3]), rng.choice([1, 2, 4]), rng.choice([1, 2, 3])
        p, t, h = (rng.choice(steps) for _ in range(3))
        places = [x + i * p for i in range(pages) for x in _values(0, page, t, kv_heads, h, dim)]
        want = base.E_SHAPE if len(set(places)) < len(places) else 0
        c = base.cache(num_pages=pages, page_size=page, kv_heads=kv_heads, head_dim=dim, page_stride=p, token_stride=t, head_stride=h)
        b = base.batch(tokens=2)
        assert lib.limits_check_append(ctypes.byref(base.append_desc(c, b, q_heads=2, rot_dim=0))) == want, (pages, page, kv_heads, p, t, h)
        assert lib.limits_check_attention(ctypes.byref(base.attention_desc(c, b, q_heads=kv_heads))) == 0
        found["cache"][want != 0] += 1
    assert min(found["rows"] + found["cache"]) > 200
    # large ones, in every order
    big = dict(num_pages=1 << 20, page_size=256, kv_heads=8, head_dim=64)
    for strides in [(256 * 512, 512, 64), (256 * 512, 64, 256 * 64), (64, (1 << 20) * 64, (1 << 28) * 64), (512, (1 << 20) * 512, 64)]:
        names = dict(zip(("page_stride", "token_stride", "head_stride"), strides))
        d = base.append_desc(base.cache(**big, **names, k=1 << 42, v=1 << 45), base.batch(), rot_dim=0)
        assert lib.limits_check_append(ctypes.byref(d)) == 0
        d = base.append_desc(base.cache(**big, **{**names, "token_stride": names["token_stride"] - 8}, k=1 << 42, v=1 << 45), base.batch(), rot_dim=0)
        assert lib.limits_check_append(ctypes.byref(d)) == base.E_SHAPE


def test_keys_and_values_of_the_cache_in_one_another(lib):
    """Pages that hold both, in any order, are appended to; a value in a key's place is refused.  Attention, which only reads, takes one tensor for both."""
    rng, dim, found = random.Random(10), 64, [0, 0]
    at = 1 << 30
    for _ in range(1500):
        pages, page, kv_heads = rng.choice([1, 2, 3]), rng.choice([1, 2, 4]), rng.choice([1, 2, 3])
        h = rng.choice([64, 128, 136])
        t = h * kv_heads * rng.choice([1, 2])
        p = t * page * rng.choice([1, 2]) + rng.choice([0, 64])
        off = 8 * rng.randint(-5, pages * p // 8 + 5) if rng.random() < 0.5 else rng.choice([64, h * kv_heads, t * page, pages * p, -64, 0])
        keys = [x + i * p for i in range(pages) for x in _values(0, page, t, kv_heads, h, dim)]
        want = not set(keys).isdisjoint(x + off for x in keys)
        c = base.cache(k=at, v=at + 2 * off, num_pages=pages, page_size=page, kv_heads=kv_heads, head_dim=dim, page_stride=p, token_stride=t, head_stride=h)
        b = base.batch(tokens=2)
        assert lib.limits_check_append(ctypes.byref(base.append_desc(c, b, q_heads=2, rot_dim=0))) == (base.E_ALIAS if want else 0), (pages, page, kv_heads, p, t, h, off)
        assert lib.limits_check_attention(ctypes.byref(base.attention_desc(c, b, q_heads=kv_heads))) == 0
        found[want] += 1
    assert min(found) > 200


def test_a_place_left_out_hides_no_wait_that_ran_out(lib):
    """Results behind a wait that ran out are worth nothing; a page number out of bounds, whenever it was found, is told only while there is no such wait."""
    assert [lib.limits_reported(w, p) for w, p in [(0, 0), (0, 0xA01), (0x701, 0), (0x701, 0xA01), (0xA10, 0xA01)]] == [0, 0xA01, 0x701, 0x701, 0xA10]
    csrc = os.path.join(ROOT, "qwen3-27b-thor-runner_b200", "csrc")
    for name in sorted(os.listdir(csrc)):
        if name.endswith((".cu", ".cuh", ".h")):
            text = open(os.path.join(csrc, name)).read()
            for line in [x for x in text.split("\n") if "kStatusPlace" in x and "constexpr" not in x]:
                assert "places = kStatusPlace;" in line, (name, line)
