"""The paged cache's calls at the ends of what they take: runs longer than a wait's limit, lengths and offsets out of bounds."""
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
