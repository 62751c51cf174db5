"""The paged cache's calls at the ends of what they take: runs longer than a wait's limit, lengths and offsets out of bounds."""
import numpy as np
import pytest
import torch

import nvfp4
import paged_reference as ref

pytestmark = pytest.mark.gpu


def test_a_call_may_take_longer_than_a_wait():
    """Every wait on the device gives up after 2e9 clocks; a prompt this long takes half as many again (74 pairs of SMs, units of 512 rows and 128 keys, 4200 clocks
    each), so that no wait may span a block's run.  The values rise with the position: a row that lacks a part of its keys has another result."""
    n, dim, page = 2_700_001, 64, 256
    h = nvfp4.Handle(0, 16 << 20)
    g = torch.Generator(device="cuda").manual_seed(1)
    pages = -(-n // page)
    q = torch.randn((n, 1, dim), device="cuda", generator=g, dtype=torch.bfloat16)
    k = torch.randn((pages, page, 1, dim), device="cuda", generator=g, dtype=torch.bfloat16)
    v = torch.randn((pages, page, 1, dim), device="cuda", generator=g, dtype=torch.bfloat16)
    v += (torch.arange(pages * page, device="cuda") * (8.0 / n)).to(torch.bfloat16).view(pages, page, 1, 1)
    out = torch.full_like(q, 7.0)
    order = torch.randperm(pages, device="cuda", generator=g).to(torch.int32)
    batch = nvfp4.PagedBatch(torch.tensor([n], dtype=torch.int32, device="cuda"), order.view(1, -1), tokens=n,
                             cu_q=torch.tensor([0, n], dtype=torch.int32, device="cuda"), max_q_len=n)
    h.paged_attention(nvfp4.KvCache(k, v), batch, q, out)
    torch.cuda.synchronize()
    assert h.device_status() == 0
    keys, values = (x[order.long()].view(-1, dim) for x in (k, v))
    for row in [0, 1, 127, 128, 1000, 99_999, n // 3, n // 2, 2 * n // 3, n - 600_000, n - 1000, n - 129, n - 2, n - 1]:
        t = keys[:row + 1].double() @ q[row, 0].double() * dim ** -0.5
        w = torch.softmax(t, 0)
        want, size = w @ values[:row + 1].double(), w @ values[:row + 1].double().abs()
        # The result's sum is held in FP32 over 8 steps of 16 keys a unit of 128, each of which may cut off 2^-23 of what is there; a thread's sum of weights over a
        # unit's 64 keys and the units, 2^-24 each; the weights and the result are rounded to BF16; scores as in the reference's bound.
        steps = row // 16 + 1
        score = 2 * (dim + 4) * 2.0 ** -23 * float((keys[:row + 1].double().abs() @ q[row, 0].double().abs()).max()) * dim ** -0.5
        tol = (steps * 2.0 ** -23 + (row // 128 + 65) * 2.0 ** -24 + ref.BF16_HALF_STEP + score + 2.0 ** -20) * size * (1 + ref.BF16_HALF_STEP) + ref.BF16_HALF_STEP * want.abs()
        assert float(((out[row, 0].double() - want).abs() / tol).max()) <= 1.0, row
    h.close()


@pytest.mark.parametrize("new", [[1, 1, 1], [40, 3, 90], [70, 1, 2, 33]])            # either kernel, and both
def test_a_length_behind_the_table_is_told(new):
    """The keys that the table holds take part, and the status says that others did not."""
    h = nvfp4.Handle(0, 16 << 20)
    c = ref.Case(new, [200 - n for n in new], 4, 2, 128, 16, seed=len(new), gate=True, pad=2)
    cache, batch = c.objects(nvfp4)
    want, tol = ref.attention(c)
    h.paged_attention(cache, batch, c.q, c.out, gate=c.gate)
    assert h.device_status() == 0 and ref.worst(c.out, want, tol) <= 1.0
    # the last sequence: 200 positions of a table of 208, and from the second call on 9 more than it has
    last = len(new) - 1
    c.kv_dev[last] = 217
    h.paged_attention(cache, batch, c.q, c.out, gate=c.gate)
    assert h.device_status() == 0xA01
    before = int(c.starts[last])
    assert ref.worst(c.out[:before], want[:before], tol[:before]) <= 1.0
    rows = slice(before, before + new[last])
    k, v = (c.by_token(x)[c.table[last].long().cuda()].flatten(0, 1)[:208].double() for x in (c.k_cache, c.v_cache))
    for i in range(new[last]):
        n = min(217 - new[last] + i + 1, 208)
        for hd in range(4):
            t = k[:n, hd // 2] @ c.q[before + i, hd].double() * 128 ** -0.5
            w = torch.softmax(t, 0)
            o, a = w @ v[:n, hd // 2], w @ v[:n, hd // 2].abs()
            sig = torch.sigmoid(c.gate[before + i, hd].double())
            score = 2 * 132 * 2.0 ** -23 * float((k[:n, hd // 2].abs() @ c.q[before + i, hd].double().abs()).max()) * 128 ** -0.5
            off = (ref.BF16_HALF_STEP + score + 2.0 ** -20) * a * sig * (1 + ref.BF16_HALF_STEP) + ref.BF16_HALF_STEP * (o * sig).abs() + 1e-30
            assert float(((c.out[before + i, hd].double() - o * sig).abs() / off).max()) <= 1.0
    assert bool((c.out[rows.stop:] == 7).all())
    h.close()


@pytest.mark.parametrize("starts", [[0, 3, 11], [-1, 3, 8], [0, 50, 90]])
@pytest.mark.parametrize("call", ["append", "few", "many"])
def test_rows_outside_the_batch_are_told(starts, call):
    h = nvfp4.Handle(0, 16 << 20)
    c = ref.Case([4, 4], [60, 30], 40 if call == "many" else 4, 2, 128, 16, seed=3)
    cache, batch = c.objects(nvfp4)
    run = (lambda: h.kv_append(cache, batch, c.q, c.k, c.v, c.out)) if call == "append" else (lambda: h.paged_attention(cache, batch, c.q, c.out))
    run()
    assert h.device_status() == 0
    c.cu_dev.copy_(torch.tensor(starts, dtype=torch.int32))
    run()
    assert h.device_status() == 0xA01
    h.close()


@pytest.mark.parametrize("dim,q_heads,kv_heads,new,past", [
    (128, 32, 8, [1] * 5, [0, 1, 40, 700, 3000]), (128, 16, 1, [1, 1], [900, 60]), (256, 24, 2, [1, 1, 1], [5, 333, 5000]), (256, 8, 1, [1, 1], [1500, 64]),
    (64, 7, 1, [1, 2, 3, 4], [50, 0, 900, 20]), (64, 24, 3, [3, 1], [128, 2000]), (256, 6, 1, [4, 1, 2], [100, 900, 2]), (128, 8, 2, [1], [40000])])
@pytest.mark.parametrize("page", [16, 5])
def test_few_tokens_round_the_result_only(dim, q_heads, kv_heads, new, past, page):
    """One rounding to BF16, that of the result.  Queries and keys are multiples of 1/4 up to 2, so that their products are exact and what is left is: a weight's two
    operands, off by 2^-16 of it; exp2 and its argument, 2^-20 and the score's own 2^-22; the tensor core's and the sums' 2^-22 of what is there for each 16 keys
    and for 64 additions at the end."""
    h = nvfp4.Handle(0, 16 << 20)
    c = ref.Case(new, past, q_heads, kv_heads, dim, page, seed=dim + q_heads)
    g = torch.Generator(device="cuda").manual_seed(dim + page)
    quarters = lambda x: x.copy_(torch.randint(-8, 9, x.shape, device="cuda", generator=g) / 4)
    quarters(c.q), quarters(c.k_cache)
    cache, batch = c.objects(nvfp4)
    h.paged_attention(cache, batch, c.q, c.out)
    torch.cuda.synchronize()
    worst = 0.0
    for s, (n, kv) in enumerate(zip(c.new, c.kv)):
        rows = slice(int(c.starts[s]), int(c.starts[s]) + n)
        k, v = c.keys(c.k_cache, s, kv), c.keys(c.v_cache, s, kv)
        hidden = torch.arange(kv, device="cuda")[None, :] > torch.arange(kv - n, kv, device="cuda")[:, None]
        for hd in range(q_heads):
            t = (c.q[rows, hd].double() @ k[:, hd * kv_heads // q_heads].T * dim ** -0.5).masked_fill(hidden, -float("inf"))
            w = torch.softmax(t, -1)
            o, a = w @ v[:, hd * kv_heads // q_heads], w @ v[:, hd * kv_heads // q_heads].abs()
            score = t.masked_fill(hidden, 0.0).abs().amax(-1, keepdim=True)
            rel = 2.0 ** -16 + 2.0 ** -20 + (2 * score + kv / 16 + 64) * 2.0 ** -22
            tol = rel * a * (1 + ref.BF16_HALF_STEP) + ref.BF16_HALF_STEP * o.abs() + 1e-30
            worst = max(worst, float(((c.out[rows, hd].double() - o).abs() / tol).max()))
    assert worst <= 1.0
    assert h.device_status() == 0
    h.close()


def _plant(c, seed):
    """Every query is aligned with two keys that it sees, which share its attention: a key left out, or counted twice, changes its result by a sixth of a value and more.
    The two lie at positions spread over all that the row sees, its first, its last and those around multiples of 16 among them."""
    rng = np.random.default_rng(seed)
    sign = torch.Generator(device="cuda").manual_seed(seed)
    c.k_cache.copy_(torch.randint(0, 2, c.k_cache.shape, device="cuda", generator=sign) * 2 - 1)
    g = c.q_heads // c.kv_heads
    for s, (n, kv) in enumerate(zip(c.new, c.kv)):
        if n == 0:
            continue
        keys = c.keys(c.k_cache, s, kv)
        see = np.arange(kv - n, kv)[:, None] + 1
        at = [(rng.random((n, c.q_heads)) * see).astype(np.int64) for _ in range(2)]
        edges = rng.integers(0, 4, (n, c.q_heads))
        near = np.clip(at[0] // 16 * 16 + rng.integers(-1, 2, at[0].shape), 0, see - 1)
        at[0] = np.choose(edges, [at[0], near, np.broadcast_to(see - 1, at[0].shape), np.zeros_like(at[0])])
        heads = torch.arange(c.q_heads, device="cuda")[None, :] // g
        both = sum(keys[torch.from_numpy(p).cuda(), heads] for p in at)
        c.q[int(c.starts[s]):int(c.starts[s]) + n] = both * (2.0 if c.dim > 64 else 4.0)


@pytest.mark.parametrize("dim,q_heads,kv_heads", [(256, 24, 2), (128, 8, 8), (128, 32, 8), (64, 20, 1)])
@pytest.mark.parametrize("page", [16, 24, 7])
def test_every_key_counts_once_in_decode(dim, q_heads, kv_heads, page):
    h = nvfp4.Handle(0, 16 << 20)
    for seed, past in enumerate([[4999], [17] * 3 + [2000, 63, 64, 65, 130, 999], list(range(100, 3100, 53))]):
        c = ref.Case([1] * len(past), past, q_heads, kv_heads, dim, page, seed=seed)
        for turn in range(6 if len(past) == 1 else 1):
            _plant(c, 10 * seed + turn)
            cache, batch = c.objects(nvfp4)
            want, tol = ref.attention(c)
            h.paged_attention(cache, batch, c.q, c.out)
            torch.cuda.synchronize()
            assert ref.worst(c.out, want, tol) <= 1.0, (seed, turn)
    assert h.device_status() == 0
    h.close()


@pytest.mark.parametrize("dim,q_heads,kv_heads,new,past", [
    (256, 24, 2, [700], [1300]), (256, 4, 4, [129, 1, 300, 2], [1, 900, 511, 40]), (128, 32, 8, [260, 1, 40], [0, 700, 2000]), (128, 6, 2, [1000], [3000]),
    (64, 12, 6, [513, 3], [255, 800]), (64, 5, 1, [128, 128, 128], [0, 128, 129])])
@pytest.mark.parametrize("page", [16, 64, 24])
def test_every_key_counts_once_in_prompts(dim, q_heads, kv_heads, new, past, page):
    h = nvfp4.Handle(0, 16 << 20)
    c = ref.Case(new, past, q_heads, kv_heads, dim, page, seed=dim + page, pad=1)
    _plant(c, dim + page)
    cache, batch = c.objects(nvfp4)
    want, tol = ref.attention(c)
    h.paged_attention(cache, batch, c.q, c.out)
    torch.cuda.synchronize()
    assert ref.worst(c.out, want, tol) <= 1.0 and h.device_status() == 0
    h.close()


@pytest.mark.parametrize("dim,q_heads,kv_heads", [(256, 12, 2), (128, 8, 2), (64, 6, 6)])
@pytest.mark.parametrize("new,past", [([1] * 7, [0, 15, 16, 90, 300, 1000, 2000]), ([150, 1, 33, 4], [10, 500, 0, 77])])
def test_rows_head_by_head(dim, q_heads, kv_heads, new, past):
    """[heads][tokens][dim]: the head's stride above the token's, for queries, gates, new keys and values and the results."""
    h = nvfp4.Handle(0, 16 << 20)
    c = ref.Case(new, past, q_heads, kv_heads, dim, 16, seed=dim, gate=True, pad=3)
    swap = lambda t: t.transpose(0, 1).contiguous().transpose(0, 1)
    for name in ("q", "gate", "k", "v", "out"):
        setattr(c, name, swap(getattr(c, name)))
    assert c.q.stride(1) > c.q.stride(0)
    cache, batch = c.objects(nvfp4)
    want, tol = ref.attention(c)
    h.paged_attention(cache, batch, c.q, c.out, gate=c.gate)
    torch.cuda.synchronize()
    assert ref.worst(c.out, want, tol) <= 1.0
    c.out.fill_(7.0)
    f = (1e4 ** (-torch.arange(0, dim, 2, dtype=torch.float64) / dim)).float().cuda()
    (want_q, q_tol), (want_k, k_tol), want_v = ref.append(c, None, None, 1e-6, f)
    h.kv_append(cache, batch, c.q, c.k, c.v, c.out, inv_freq=f)
    torch.cuda.synchronize()
    assert ref.worst(c.out, want_q, q_tol) <= 1.0 and ref.worst(c.k_cache, want_k, k_tol) <= 1.0 and torch.equal(c.v_cache.double(), want_v)
    assert h.device_status() == 0
    h.close()
