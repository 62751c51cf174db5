"""The paged cache on a GPU: append and attention against their definitions in 64 bits, over head layouts, lengths, page sizes and orders, strides,
padded batches, bad pages, captured calls and streams."""
import numpy as np
import pytest
import torch

import nvfp4
import paged_reference as ref

pytestmark = pytest.mark.gpu
EPS = 1e-6


@pytest.fixture(scope="module")
def handle():
    h = nvfp4.Handle(0, 16 << 20)
    yield h
    torch.cuda.synchronize()
    assert h.device_status() == 0
    h.close()


def freq(rot, theta=1e7):
    return (theta ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)).float().cuda() if rot else None


def weights(dim, seed):
    g = torch.Generator().manual_seed(seed)
    return [(0.3 * torch.randn(dim, generator=g)).to(torch.bfloat16).cuda() for _ in range(2)]


def check_attention(handle, c, scale=None, times=1, **kw):
    cache, batch = c.objects(nvfp4)
    want, tol = ref.attention(c, scale=scale, **kw)
    first = None
    for _ in range(times):
        c.out.fill_(7.0)
        handle.paged_attention(cache, batch, c.q, c.out, gate=c.gate, scale=scale or 0.0)
        torch.cuda.synchronize()
        assert ref.worst(c.out, want, tol) <= 1.0
        first = c.out.clone() if first is None else first
        assert torch.equal(first, c.out)               # no order of arrival in the bits


def check_append(handle, c, q_norm, k_norm, inv_freq, positions=None, in_place=False):
    cache, batch = c.objects(nvfp4)
    (want_q, q_tol), (want_k, k_tol), want_v = ref.append(c, q_norm, k_norm, EPS, inv_freq if inv_freq is not None else torch.zeros(0, device="cuda"), positions)
    out = c.q if in_place else c.out
    if in_place:
        covered = q_tol > 0
        want_q = torch.where(covered, want_q, c.q.double())
    handle.kv_append(cache, batch, c.q, c.k, c.v, out, q_norm=q_norm, k_norm=k_norm, norm_eps=EPS, inv_freq=inv_freq, positions=positions)
    torch.cuda.synchronize()
    assert ref.worst(out, want_q, q_tol) <= 1.0
    assert ref.worst(c.k_cache, want_k, k_tol) <= 1.0
    assert torch.equal(c.v_cache.double(), want_v)


# ---------------------------------------------------------------- append

@pytest.mark.parametrize("dim,q_heads,kv_heads,rot,norm,page,order,new,past,pad", [
    (256, 24, 2, 64, True, 16, "token", [1], [777], 0),
    (256, 24, 2, 64, True, 16, "token", [1] * 5, [0, 15, 16, 31, 4000], 3),
    (256, 8, 4, 256, True, 24, "head", [3, 0, 17, 1], [5, 9, 0, 40], 2),
    (128, 32, 8, 128, False, 16, "token", [1] * 20, list(range(20)), 0),
    (128, 5, 5, 32, True, 1, "head", [7, 1], [0, 3], 1),
    (128, 6, 1, 0, True, 7, "token", [33], [100], 0),
    (64, 16, 4, 16, True, 64, "token", [65, 2], [63, 0], 5),
    (64, 3, 3, 64, False, 5, "head", [1, 1, 4], [0, 4, 5], 0),
    (256, 24, 2, 64, True, 64, "token", [400, 1, 77], [1000, 3, 0], 7),       # a block per token
])
def test_append(handle, dim, q_heads, kv_heads, rot, norm, page, order, new, past, pad):
    c = ref.Case(new, past, q_heads, kv_heads, dim, page, seed=dim + page, order=order, pad=pad, lead=1 if pad else 0)
    qn, kn = weights(dim, 3) if norm else (None, None)
    check_append(handle, c, qn, kn, freq(rot))


def test_append_one_token_per_sequence_without_cu_q(handle):
    c = ref.Case([1] * 9, list(range(0, 90, 10)), 4, 2, 128, 16, seed=5, cu=False, pad=4)
    check_append(handle, c, *weights(128, 1), freq(128))


def test_append_in_place_and_from_a_merged_projection(handle):
    """q interleaved with its gate, k and v behind it in the same rows; q normed and rotated where it lies."""
    c = ref.Case([5, 1, 30], [11, 500, 0], 6, 2, 256, 16, seed=8, pad=2)
    merged = torch.randn((c.rows, (2 * 6 + 2 * 2) * 256), generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).cuda()
    before = merged.clone()
    qg = merged[:, :12 * 256].view(c.rows, 6, 512)
    c.q = qg[..., :256]
    c.k, c.v = merged[:, 12 * 256:14 * 256].view(c.rows, 2, 256), merged[:, 14 * 256:].view(c.rows, 2, 256)
    check_append(handle, c, *weights(256, 2), freq(64), in_place=True)
    assert torch.equal(merged[:, 12 * 256:], before[:, 12 * 256:]) and torch.equal(qg[..., 256:], before[:, :12 * 256].view(c.rows, 6, 512)[..., 256:])


def test_append_without_queries(handle):
    c = ref.Case([4, 1], [0, 20], 2, 2, 128, 16, seed=9)
    cache, batch = c.objects(nvfp4)
    _, (want_k, k_tol), want_v = ref.append(c, None, weights(128, 4)[1], EPS, freq(32))
    handle.kv_append(cache, batch, None, c.k, c.v, None, k_norm=weights(128, 4)[1], norm_eps=EPS, inv_freq=freq(32))
    torch.cuda.synchronize()
    assert ref.worst(c.k_cache, want_k, k_tol) <= 1.0 and torch.equal(c.v_cache.double(), want_v) and bool((c.out == 7).all())


def test_append_given_and_far_positions(handle):
    """The angle of position 2^31 - 1 and of some in front of it: in FP32 it would be off by up to 128 radians."""
    c = ref.Case([6], [2], 4, 2, 128, 16, seed=10)
    positions = torch.tensor([2147483647, 16777217, 0, 1000003, 131071, 5], dtype=torch.int32, device="cuda")
    check_append(handle, c, *weights(128, 5), freq(128), positions=positions)


def test_append_leaves_out_padded_sequences_and_bad_places():
    h = nvfp4.Handle(0, 16 << 20)
    c = ref.Case([1, 1, 2, 1], [40, 7, 14, 3], 4, 2, 128, 16, seed=11)
    c.kv_dev[1] = 0                                    # padded: no position
    c.table_dev[2, 0] = c.num_pages                    # bad for position 14 and 15
    c.table_dev[3, 0] = -1
    k0, v0 = c.k_cache.clone(), c.v_cache.clone()
    cache, batch = c.objects(nvfp4)
    h.kv_append(cache, batch, c.q, c.k, c.v, c.out, inv_freq=freq(128))
    torch.cuda.synchronize()
    page, slot = int(c.table[0, 2]), 40 % 16
    k0[page, slot], v0[page, slot] = c.k_cache[page, slot], c.v[0]
    assert torch.equal(c.k_cache, k0) and torch.equal(c.v_cache, v0)
    assert bool((c.out[1] == 7).all()) and not bool((c.out[[0, 2, 3, 4]] == 7).all(-1).any())
    assert h.device_status() == 0xA01
    h.close()


# ---------------------------------------------------------------- attention

LAYOUTS = [(256, 24, 2), (256, 4, 4), (128, 32, 8), (128, 6, 2), (128, 16, 1), (64, 5, 1), (64, 12, 6), (64, 40, 2)]


@pytest.mark.parametrize("dim,q_heads,kv_heads", LAYOUTS)
@pytest.mark.parametrize("page,order", [(16, "token"), (64, "head"), (24, "token"), (1, "head")])
def test_decode(handle, dim, q_heads, kv_heads, page, order):
    """One new token: lengths of one, around a page and a unit's 64 and 128 tokens, and long enough to be split."""
    past = [0, 1, 14, 15, 16, 62, 63, 64, 126, 127, 128, 129, 1000, 2500]
    c = ref.Case([1] * len(past), past, q_heads, kv_heads, dim, page, seed=dim + page, order=order, gate=page == 16, pad=page % 3)
    check_attention(handle, c, times=2)


@pytest.mark.parametrize("past", [0, 5, 700, 9001, 40000])
@pytest.mark.parametrize("dim,q_heads,kv_heads", [(256, 24, 2), (128, 8, 8), (64, 3, 1)])
def test_decode_of_one_sequence(handle, past, dim, q_heads, kv_heads):
    c = ref.Case([1], [past], q_heads, kv_heads, dim, 16, seed=past, gate=True)
    check_attention(handle, c, times=3)


@pytest.mark.parametrize("sequences", [149, 700])
def test_decode_of_many_sequences(handle, sequences):
    rng = np.random.default_rng(sequences)
    c = ref.Case([1] * sequences, [int(x) for x in np.exp(rng.uniform(0, np.log(600), sequences))], 4, 2, 128, 16, seed=1, cu=False, pad=3)
    check_attention(handle, c)


@pytest.mark.parametrize("dim,q_heads,kv_heads", LAYOUTS)
def test_few_tokens(handle, dim, q_heads, kv_heads):
    """Several new tokens: each row its own last key, tiles of 16 rows that end inside a token's heads, sequences without new tokens."""
    c = ref.Case([4, 2, 0, 8, 3, 1], [0, 100, 50, 15, 1000, 333], q_heads, kv_heads, dim, 16, seed=dim, gate=True, pad=2)
    check_attention(handle, c, times=2)


@pytest.mark.parametrize("dim,q_heads,kv_heads", LAYOUTS)
@pytest.mark.parametrize("page,order", [(16, "token"), (64, "head"), (128, "token"), (256, "token"), (40, "token")])
def test_prompts(handle, dim, q_heads, kv_heads, page, order):
    """Prompts, chunks behind a past, and single tokens in the same batch; lengths around 128."""
    c = ref.Case([129, 1, 128, 37, 300, 1, 0, 127], [0, 260, 128, 77, 1, 0, 5, 512], q_heads, kv_heads, dim, page, seed=dim + page, order=order, gate=page == 64, pad=3)
    check_attention(handle, c, times=2)


def test_one_long_prompt(handle):
    c = ref.Case([1500], [700], 12, 2, 256, 32, seed=4, gate=True)
    check_attention(handle, c, times=2)


def test_strided_rows_and_scale(handle):
    c = ref.Case([3, 1, 40], [10, 90, 0], 6, 2, 128, 16, seed=6)
    g = torch.Generator().manual_seed(2)
    qg = torch.randn((c.rows, 6, 256 + 8), generator=g).to(torch.bfloat16).cuda()
    c.q, c.gate = qg[..., :128], qg[..., 128:256]
    wide = torch.full((c.rows, 6, 136), 7.0, dtype=torch.bfloat16, device="cuda")
    c.out = wide[..., :128]
    check_attention(handle, c, scale=0.21)
    assert bool((wide[..., 128:] == 7).all())
    check_attention(handle, c, scale=-0.1)


@pytest.mark.parametrize("new", [1, 3, 50, 200])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -3e38])
def test_slots_behind_a_sequence_may_hold_anything(handle, new, value):
    c = ref.Case([new, new], [37, 130], 8, 2, 128, 64, seed=new, table_extra=2)
    for cache in (c.k_cache, c.v_cache):
        held = torch.zeros(cache.shape[:2], dtype=torch.bool, device="cuda")
        for s, kv in enumerate(c.kv):
            for p in range(kv):
                held[int(c.table[s, p // 64]), p % 64] = True
        cache[~held] = value
    check_attention(handle, c)


def test_rows_that_see_nothing_are_zero(handle):
    c = ref.Case([1, 4, 200, 1], [20, 0, 0, 9], 4, 2, 128, 16, seed=12, gate=True)
    c.kv_dev[0] = 0
    c.kv_dev[1] = 2                                    # two of its four rows stand in front of position 0
    c.kv_dev[2] = 60
    cache, batch = c.objects(nvfp4)
    handle.paged_attention(cache, batch, c.q, c.out, gate=c.gate)
    torch.cuda.synchronize()
    assert bool((c.out[0] == 0).all()) and bool((c.out[1:3] == 0).all()) and bool((c.out[5:145] == 0).all())
    assert not bool((c.out[3:5] == 0).all(-1).any()) and not bool((c.out[145:205] == 0).all(-1).any())
    want, tol = ref.attention(c)
    assert ref.worst(c.out[205:], want[205:], tol[205:]) <= 1.0


@pytest.mark.parametrize("new", [1, 5, 150])
def test_bad_pages_take_part_in_nothing(new):
    """The result is that of the tokens whose pages are in bounds, and the status says that some were not."""
    h = nvfp4.Handle(0, 16 << 20)
    c = ref.Case([new], [200], 4, 2, 128, 16, seed=13)
    good = [p for p in range(c.kv[0]) if p // 16 not in (1, 7)]
    want = torch.zeros_like(c.out, dtype=torch.float64)
    k, v = c.keys(c.k_cache, 0, c.kv[0])[good], c.keys(c.v_cache, 0, c.kv[0])[good]
    for i in range(new):
        seen = torch.tensor(good, device="cuda") <= 200 + i
        for hd in range(4):
            t = (k[:, hd // 2] @ c.q[i, hd].double()) * 128 ** -0.5
            want[i, hd] = torch.softmax(t.masked_fill(~seen, -float("inf")), 0) @ v[:, hd // 2]
    c.table_dev[0, 1], c.table_dev[0, 7] = c.num_pages, -7
    cache, batch = c.objects(nvfp4)
    h.paged_attention(cache, batch, c.q, c.out)
    torch.cuda.synchronize()
    assert float((c.out.double() - want).norm() / want.norm()) < 5e-3
    assert h.device_status() == 0xA01
    h.close()


def test_offsets_beyond_32_bits(handle):
    """Pages 2^30 elements apart, and slots, so that the last ones lie behind 2^31 elements."""
    stride = 1 << 30
    buf = [torch.zeros(2 * stride + (1 << 20), dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    c = ref.Case([3, 140], [60, 4], 4, 2, 128, 64, seed=14)
    assert c.num_pages >= 4
    c.table = torch.tensor([[2, 0, 0], [1, 0, 2]], dtype=torch.int32)       # the sequences share what only the second one may be long enough for
    c.kv, c.past = [63, 144], [60, 4]
    c.table_dev = c.table.cuda()
    c.num_pages = 3
    views = [b.as_strided((3, 64, 2, 128), (stride, 512, 128, 1)) for b in buf]
    for view, src in zip(views, (c.k_cache, c.v_cache)):
        view.copy_(src[:3])
    c.k_cache, c.v_cache = views
    check_attention(handle, c)
    c2 = ref.Case([1, 70], [62, 0], 4, 2, 128, 64, seed=15)
    c2.table, c2.num_pages, c2.k_cache, c2.v_cache = torch.tensor([[2, 0], [1, 0]], dtype=torch.int32), 3, views[0], views[1]
    c2.table_dev = c2.table.cuda()
    check_append(handle, c2, *weights(128, 6), freq(128))


# ---------------------------------------------------------------- as they are used

def _run_layer(handle, c, qn, kn, f, out_q, stream=None):
    cache, batch = c.objects(nvfp4)
    handle.kv_append(cache, batch, c.q, c.k, c.v, out_q, q_norm=qn, k_norm=kn, norm_eps=EPS, inv_freq=f, stream=stream)
    handle.paged_attention(cache, batch, out_q, c.out, gate=c.gate, stream=stream)


@pytest.mark.parametrize("dim,q_heads,kv_heads,rot", [(256, 24, 2, 64), (128, 8, 2, 128), (64, 4, 4, 32)])
def test_a_sequence_token_by_token_is_the_prompt_at_once(handle, dim, q_heads, kv_heads, rot):
    """A prompt, then tokens one and several at a time, back to back on a stream; every row is what one call over all of them gives, up to the
    rounding of weights and results."""
    total, pieces = 230, [150, 1, 1, 5, 1, 40, 1, 1, 30]
    c = ref.Case([total], [0], q_heads, kv_heads, dim, 16, seed=20, gate=True)
    qn, kn = weights(dim, 7)
    f = freq(rot)
    _run_layer(handle, c, qn, kn, f, torch.empty_like(c.q))
    torch.cuda.synchronize()
    whole, keys, values = c.out.clone(), c.k_cache.clone(), c.v_cache.clone()
    c.k_cache.fill_(float("nan"))
    c.v_cache.fill_(float("nan"))
    at, outs = 0, []
    for n in pieces:
        d = ref.Case([n], [at], q_heads, kv_heads, dim, 16, seed=21, gate=True)
        d.table, d.table_dev, d.num_pages = c.table, c.table_dev, c.num_pages
        d.k_cache, d.v_cache = c.k_cache, c.v_cache
        d.q, d.k, d.v, d.gate = c.q[at:at + n], c.k[at:at + n], c.v[at:at + n], c.gate[at:at + n]
        _run_layer(handle, d, qn, kn, f, torch.empty_like(d.q))
        outs.append(d.out)
        at += n
    torch.cuda.synchronize()
    got = torch.cat(outs)
    held = ~torch.isnan(c.k_cache.float())
    assert torch.equal(c.k_cache[held], keys[held]) and torch.equal(c.v_cache[held], values[held]) and int(held.sum()) == total * kv_heads * dim
    # two results that are each half a step of weights and result from the exact one
    assert float((got.double() - whole.double()).norm() / whole.double().norm()) <= 4 * ref.BF16_HALF_STEP


def test_captured_step_replayed_with_other_lengths(handle):
    """Append and attention of a padded batch captured once; replays with other lengths, tables and rows give the bits of eager calls."""
    most, dim, hq, hk = 12, 128, 8, 2
    cases = [ref.Case([1] * n, past, hq, hk, dim, 16, seed=30 + n, gate=True, pad=most - n)
             for n, past in [(12, [3] * 12), (5, [0, 900, 15, 16, 2000]), (1, [5000]), (9, [100] * 9)]]
    cols, pages = max(c.table.shape[1] for c in cases), max(c.num_pages for c in cases)
    fixed = ref.Case([1] * most, [0] * most, hq, hk, dim, 16, seed=40, gate=True, spare=pages)
    fixed.table_dev = torch.zeros((most, cols), dtype=torch.int32, device="cuda")
    fixed.table = fixed.table_dev.cpu()
    qn, kn = weights(dim, 8)
    f, out_q = freq(dim), torch.empty_like(fixed.q)

    def fill(c):
        n = len(c.new)
        fixed.k_cache[:c.num_pages], fixed.v_cache[:c.num_pages] = c.k_cache, c.v_cache
        for name in ("q", "k", "v", "gate"):
            getattr(fixed, name).copy_(getattr(c, name))
        fixed.cu_dev.copy_(torch.tensor(list(c.starts) + [n] * (most - n), dtype=torch.int32))
        fixed.kv_dev.copy_(torch.tensor(c.kv + [0] * (most - n), dtype=torch.int32))
        fixed.table_dev.zero_()
        fixed.table_dev[:n, :c.table.shape[1]] = c.table_dev
        fixed.out.fill_(7.0)

    want = []
    for c in cases:
        fill(c)
        _run_layer(handle, fixed, qn, kn, f, out_q)
        torch.cuda.synchronize()
        want.append((fixed.out.clone(), fixed.k_cache.clone()))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        _run_layer(handle, fixed, qn, kn, f, out_q)
    for r in range(24):
        i = r * 3 % len(cases)
        fill(cases[i])
        graph.replay()
        torch.cuda.synchronize()
        n = cases[i].num_pages                             # the pages behind hold what the batches before left
        same = torch.equal(fixed.out, want[i][0]), torch.equal(fixed.k_cache[:n], want[i][1][:n])
        assert same == (True, True), r
        assert bool((fixed.out[len(cases[i].new):] == 7).all())


def test_on_another_stream_behind_a_kernel_that_writes_the_inputs(handle):
    c = ref.Case([1] * 8, [1000 + i for i in range(8)], 8, 2, 256, 16, seed=50, gate=True)
    want, tol = ref.attention(c)
    cache, batch = c.objects(nvfp4)
    q, k, v, kv = c.q.clone(), c.k_cache.clone(), c.v_cache.clone(), c.kv_dev.clone()
    s = torch.cuda.Stream()
    big = torch.zeros(1 << 26, device="cuda")
    for _ in range(5):
        for t in (c.q, c.k_cache, c.v_cache, c.kv_dev):
            t.zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(s):
            big.add_(1.0)
            for t, x in ((c.k_cache, k), (c.v_cache, v), (c.q, q), (c.kv_dev, kv)):
                t.copy_(x)
            handle.paged_attention(cache, batch, c.q, c.out, gate=c.gate)
        torch.cuda.synchronize()
        assert ref.worst(c.out, want, tol) <= 1.0


def test_launches_are_counted(handle):
    c = ref.Case([1], [10], 4, 2, 128, 16, seed=60)
    before = handle.launch_count()
    _run_layer(handle, c, None, None, None, torch.empty_like(c.q))
    assert handle.launch_count() >= before + 2
    c.rows = 0
    cache, batch = c.objects(nvfp4)
    before = handle.launch_count()
    handle.paged_attention(cache, batch, c.q, c.out)       # no rows: nothing to do
    assert handle.launch_count() == before


# ---------------------------------------------------------------- what no ordinary batch brings together

FEW_AND_MANY = [[1] * 6, [1, 3, 4, 2], [90, 1, 260], [33]]      # new tokens: either kernel, and both


@pytest.mark.parametrize("dim,q_heads,kv_heads", [(256, 12, 2), (128, 16, 4), (64, 6, 2)])
@pytest.mark.parametrize("new", FEW_AND_MANY)
def test_gates_of_any_size(handle, dim, q_heads, kv_heads, new):
    """Far beyond what the exponential holds, in either direction, beside ordinary ones: -inf closes, inf opens."""
    c = ref.Case(new, [3000] + [40] * (len(new) - 1), q_heads, kv_heads, dim, 16, seed=dim + len(new), gate=True)
    g = torch.Generator().manual_seed(3)
    far = torch.tensor([-float("inf"), float("inf"), -43.5, -43.75, -60.0, -87.0, -120.0, -3e38, 60.0, 3e38]).to(torch.bfloat16)
    pick = torch.randint(0, 4 * len(far), c.gate.shape, generator=g)
    c.gate = torch.where(pick.cuda() < len(far), far.cuda()[pick.cuda() % len(far)], c.gate)
    check_attention(handle, c)


@pytest.mark.parametrize("dim,q_heads,kv_heads", [(256, 12, 2), (128, 16, 4), (64, 6, 2)])
@pytest.mark.parametrize("new", FEW_AND_MANY)
def test_nan_stays_with_its_query_and_its_gate(handle, dim, q_heads, kv_heads, new):
    c = ref.Case(new, [9000] + [40] * (len(new) - 1), q_heads, kv_heads, dim, 16, seed=dim + len(new), gate=True)
    want, tol = ref.attention(c)
    row, r2 = c.rows // 2, c.rows - 1
    c.q[row, 1, 5] = c.q[0, q_heads - 1, 0] = float("nan")
    c.gate[r2, 0, 3] = c.gate[r2, 2, 8] = float("nan")
    nan = torch.zeros_like(tol, dtype=torch.bool)
    nan[row, 1] = nan[0, q_heads - 1] = nan[r2, 0, 3] = nan[r2, 2, 8] = True
    cache, batch = c.objects(nvfp4)
    handle.paged_attention(cache, batch, c.q, c.out, gate=c.gate)
    torch.cuda.synchronize()
    assert torch.equal(torch.isnan(c.out), nan)
    assert ref.worst(torch.where(nan, 0, c.out), torch.where(nan, 0, want), tol) <= 1.0


@pytest.mark.parametrize("page", [1, 4, 8, 12, 16, 64])
@pytest.mark.parametrize("dim,q_heads,kv_heads", [(256, 6, 1), (128, 4, 2), (64, 3, 3)])
@pytest.mark.parametrize("new", [1, 2, 40])
def test_whole_units_without_a_page_behind_values_of_nan(page, dim, q_heads, kv_heads, new):
    """Every second sequence has values of NaN, which stay behind in shared memory; the others lack pages for more tokens than a unit holds, in
    front, in the middle and at the end.  Theirs is the attention over the pages that are there."""
    h = nvfp4.Handle(0, 16 << 20)
    n, length = 120 if new < 40 else 12, 400
    c = ref.Case([new] * n, [length - new] * n, q_heads, kv_heads, dim, page, seed=page)
    gone = torch.zeros(length, dtype=torch.bool)
    for s in range(n):
        if s % 2 == 0:
            c.v_cache[c.table[s].long().cuda()] = float("nan")
            continue
        first = [0, 96, 208][s // 2 % 3]
        entries = range(-(-first // page), -(-first // page) + 192 // page)
        for e in entries:
            c.table_dev[s, e] = [-1, c.num_pages][e % 2]
    cache, batch = c.objects(nvfp4)
    h.paged_attention(cache, batch, c.q, c.out)
    torch.cuda.synchronize()
    out = c.out.view(n, new, q_heads, dim)
    assert bool(torch.isnan(out[0::2]).all()) and bool(torch.isfinite(out[1::2]).all())
    assert h.device_status() == 0xA01
    g = q_heads // kv_heads
    for s in (1, 3, 5, n - 1):
        there = ((c.table_dev[s] >= 0) & (c.table_dev[s] < c.num_pages)).repeat_interleave(page)[:length]
        k, v = c.keys(c.k_cache, s, length).cuda(), c.keys(c.v_cache, s, length).cuda()
        seen = there[None, :] & (torch.arange(length, device="cuda")[None, :] <= torch.arange(length - new, length, device="cuda")[:, None])
        for hd in range(q_heads):
            t = (c.q[s * new:(s + 1) * new, hd].double() @ k[:, hd // g].T * dim ** -0.5).masked_fill(~seen, -float("inf"))
            w = torch.softmax(t, -1)
            want, size = w @ v[:, hd // g], w @ v[:, hd // g].abs()
            tol = 2 * ref.BF16_HALF_STEP * size + 1e-5 * size + ref.BF16_HALF_STEP * want.abs() + 1e-30
            assert ref.worst(out[s, :, hd], want, tol) <= 1.0
    h.close()


@pytest.mark.parametrize("dim,q_heads,kv_heads,new", [(256, 12, 2, 11), (256, 2, 2, 40), (128, 16, 4, 40), (128, 8, 8, 5), (64, 6, 1, 300), (64, 4, 2, 17)])
def test_few_tokens_behind_a_very_long_past(handle, dim, q_heads, kv_heads, new):
    """An item whose parts are more than a join has under way at once."""
    c = ref.Case([new], [30011], q_heads, kv_heads, dim, 64, seed=dim + new, gate=dim == 256)
    check_attention(handle, c, times=2)


@pytest.mark.parametrize("dim,q_heads,kv_heads", [(256, 24, 2), (128, 32, 8), (64, 40, 2)])
def test_rows_around_the_border_of_the_two_kernels(handle, dim, q_heads, kv_heads):
    """Sequences of one to forty rows in one call, each by the kernel for its own."""
    new = [1, 2, 3, 4, 5, 7, 8, 9, 16, 17, 1, 32, 33, 40]
    c = ref.Case(new, [(i * 977) % 3000 for i in range(len(new))], q_heads, kv_heads, dim, 16, seed=dim, pad=3, lead=2, gate=True)
    check_attention(handle, c)


@pytest.mark.parametrize("hint", [1, 2, 50, 100000])
def test_the_longest_run_may_be_guessed_wrong(handle, hint):
    c = ref.Case([70, 1, 30, 2], [100, 900, 0, 33], 8, 2, 128, 16, seed=hint, pad=5)
    cache, _ = c.objects(nvfp4)
    want, tol = ref.attention(c)
    handle.paged_attention(cache, nvfp4.PagedBatch(c.kv_dev, c.table_dev, tokens=c.rows, cu_q=c.cu_dev, max_q_len=hint), c.q, c.out)
    torch.cuda.synchronize()
    assert ref.worst(c.out, want, tol) <= 1.0


def test_more_heads_in_a_group_than_a_tile_has_rows(handle):
    c = ref.Case([3, 1, 40], [50, 700, 9], 130, 1, 64, 16, seed=4)
    check_attention(handle, c)
    c = ref.Case([3, 1, 40], [50, 700, 9], 128, 1, 128, 16, seed=5, gate=True)
    check_attention(handle, c)


@pytest.mark.parametrize("new", [1, 60])
def test_sequences_that_share_a_prefix(handle, new):
    c = ref.Case([new] * 5, [512] * 5, 8, 2, 128, 32, seed=6)
    c.table[1:, :16] = c.table[0, :16]
    c.table_dev = c.table.cuda()
    check_attention(handle, c)


def test_two_handles_on_two_streams_at_once():
    handles = [nvfp4.Handle(0, 16 << 20) for _ in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    cases = [ref.Case([200, 1, 3], [4000, 9000, 50], 12, 2, 256, 16, seed=s, gate=True) for s in (1, 2)]
    torch.cuda.synchronize()
    for _ in range(4):
        for h, s, c in zip(handles, streams, cases):
            with torch.cuda.stream(s):
                h.paged_attention(*c.objects(nvfp4), c.q, c.out, gate=c.gate)
    torch.cuda.synchronize()
    for h, c in zip(handles, cases):
        want, tol = ref.attention(c)
        assert ref.worst(c.out, want, tol) <= 1.0 and h.device_status() == 0
        h.close()


def test_calls_behind_one_another_share_the_scratch(handle):
    """Different batches, kernels and head sizes through one handle without a wait in between."""
    cases = [ref.Case(n, p, q, k, d, 16, seed=i) for i, (n, p, q, k, d) in enumerate([
        ([1], [20000], 12, 2, 256), ([300], [5000], 8, 2, 128), ([1] * 40, [700] * 40, 4, 4, 64), ([500, 1], [0, 9000], 6, 1, 256), ([1] * 3, [5000] * 3, 16, 2, 128)])]
    torch.cuda.synchronize()
    for _ in range(3):
        for c in cases:
            handle.paged_attention(*c.objects(nvfp4), c.q, c.out)
    torch.cuda.synchronize()
    for c in cases:
        want, tol = ref.attention(c)
        assert ref.worst(c.out, want, tol) <= 1.0


def test_nothing_to_do(handle):
    c = ref.Case([0, 0], [5, 9], 4, 2, 128, 16, seed=1, pad=4)
    cache, batch = c.objects(nvfp4)
    handle.paged_attention(cache, batch, c.q, c.out)
    k = c.k_cache.clone()
    handle.kv_append(cache, batch, c.q, c.k, c.v, c.out)
    torch.cuda.synchronize()
    assert bool((c.out == 7).all()) and torch.equal(c.k_cache, k)


@pytest.mark.parametrize("dim,q_heads,kv_heads,new", [(256, 24, 2, 2), (256, 12, 4, 9), (256, 6, 1, 5), (128, 32, 8, 8), (128, 6, 2, 7), (128, 17, 1, 1), (64, 16, 4, 6), (64, 20, 1, 1),
                                                      (64, 32, 1, 1)])
@pytest.mark.parametrize("page", [16, 24, 5])
def test_rows_of_two_tiles(handle, dim, q_heads, kv_heads, new, page):
    """17 to 32 rows a sequence, from one key to parts in many blocks; with and without gates, the second tile full or with a row or two."""
    past = [0, 3, 31, 32, 33, 63, 64, 127, 500, 3000, 9000]
    c = ref.Case([new, max(new - 1, 1)] + [new] * (len(past) - 2), past, q_heads, kv_heads, dim, page, seed=dim + new, gate=page == 16, pad=2)
    check_attention(handle, c, times=2)


@pytest.mark.parametrize("dim,q_heads,kv_heads,new", [(256, 24, 2, 2), (128, 32, 8, 8), (64, 20, 1, 1)])
def test_two_tiles_of_one_long_sequence(handle, dim, q_heads, kv_heads, new):
    c = ref.Case([new], [40000], q_heads, kv_heads, dim, 32, seed=dim, gate=True)
    check_attention(handle, c, times=2)
