"""Batches over a paged cache for the tests, and the operators on them from their definitions in 64 bits."""
import numpy as np
import torch

BF16_HALF_STEP = torch.finfo(torch.bfloat16).eps / 2      # 2^-8, relative


class Case:
    """Sequences with `new` new tokens behind `past` ones, pages in a random order, everything a function of the seed."""

    def __init__(self, new, past, q_heads, kv_heads, dim, page, seed=0, order="token", pad=0, gate=False, cu=True, spare=2, device="cuda", table_extra=0, lead=0):
        g = torch.Generator().manual_seed(seed)
        normal = lambda *s: torch.randn(s, generator=g).to(torch.bfloat16).to(device)
        self.new, self.past, self.q_heads, self.kv_heads, self.dim, self.page = new, past, q_heads, kv_heads, dim, page
        self.kv = [n + p for n, p in zip(new, past)]
        pages = [max(0, -(-k // page)) for k in self.kv]
        self.num_pages = sum(pages) + spare
        cols = max(max(pages), 1) + table_extra
        perm = torch.randperm(self.num_pages, generator=g).to(torch.int32)
        self.table = torch.full((len(new), cols), -1 if table_extra else 0, dtype=torch.int32)
        at = 0
        for s, n in enumerate(pages):
            self.table[s, :n] = perm[at:at + n]
            at += n
        self.free_pages = perm[at:].tolist()
        self.starts = np.concatenate([[0], np.cumsum(new)]).astype(np.int32) + lead
        self.rows = int(self.starts[-1]) + pad
        shape = (self.num_pages, page, kv_heads, dim) if order == "token" else (self.num_pages, kv_heads, page, dim)
        self.k_cache, self.v_cache, self.order = normal(*shape), normal(*shape), order
        self.q = normal(self.rows, q_heads, dim) * 2
        self.gate = normal(self.rows, q_heads, dim) if gate else None
        self.k, self.v = normal(self.rows, kv_heads, dim), normal(self.rows, kv_heads, dim)
        self.out = torch.full((self.rows, q_heads, dim), 7.0, dtype=torch.bfloat16, device=device)
        self.cu_dev = torch.from_numpy(self.starts).to(device) if cu else None
        self.kv_dev = torch.tensor(self.kv, dtype=torch.int32, device=device)
        self.table_dev = self.table.to(device)

    def objects(self, nvfp4):
        cache = nvfp4.KvCache(self.k_cache, self.v_cache, order=self.order)
        return cache, nvfp4.PagedBatch(self.kv_dev, self.table_dev, tokens=self.rows, cu_q=self.cu_dev, max_q_len=max(self.new) if self.new else 1)

    def by_token(self, cache):
        """The cache as [pages, page, heads, dim]."""
        return cache if self.order == "token" else cache.transpose(1, 2)

    def keys(self, cache, s, n):
        t = self.table[s, :-(-n // self.page)].long().to(cache.device)
        return self.by_token(cache)[t].flatten(0, 1)[:n].double()


def attention(c, scale=None, k_cache=None, v_cache=None):
    """(expected rows, how far each value may be off): weights rounded to BF16 (half a step of each, so of sum w|v|), the result rounded
    to BF16, and scores whose sums of dim products are held in FP32: each of dim + 4 additions is off by at most 2^-23 of the sum of the products'
    magnitudes (the tensor core truncates), which moves a weight, and the sum of all, by that relative to themselves; 2^-20 for exp2, sigmoid and the
    division."""
    k_cache, v_cache = c.k_cache if k_cache is None else k_cache, c.v_cache if v_cache is None else v_cache
    scale = c.dim ** -0.5 if scale is None else scale
    want, tol = c.out.double().clone(), torch.zeros(c.out.shape, dtype=torch.float64, device=c.out.device)
    g = c.q_heads // c.kv_heads
    for s, (n, kv) in enumerate(zip(c.new, c.kv)):
        rows = slice(int(c.starts[s]), int(c.starts[s]) + n)
        if n == 0:
            continue
        k, v = c.keys(k_cache, s, kv).to(c.out.device), c.keys(v_cache, s, kv).to(c.out.device)
        hidden = torch.arange(kv, device=c.out.device)[None, :] > torch.arange(kv - n, kv, device=c.out.device)[:, None]
        q = c.q[rows].double()
        for h in range(c.q_heads):
            kh, vh = k[:, h // g], v[:, h // g]
            t = q[:, h] @ kh.T * scale
            size = ((q[:, h].abs() @ kh.abs().T) * abs(scale)).masked_fill(hidden, 0.0).amax(-1, keepdim=True) if kv else torch.zeros(n, 1, device=c.out.device)
            t = t.masked_fill(hidden, -float("inf"))
            w = torch.exp(t - t.amax(-1, keepdim=True)) if kv else t
            w = torch.nan_to_num(w / w.sum(-1, keepdim=True))
            o, a = w @ vh, w @ vh.abs()
            rel = 2 * (c.dim + 4) * 2.0 ** -23 * size + 2.0 ** -20
            err = (BF16_HALF_STEP + rel) * a
            if c.gate is not None:
                sig = torch.sigmoid(c.gate[rows, h].double())
                o, err = o * sig, err * sig
            want[rows, h] = o
            tol[rows, h] = err * (1 + BF16_HALF_STEP) + BF16_HALF_STEP * o.abs() + 1e-30
    return want, tol


def normed(x, w, eps):
    x = x.double()
    return x if w is None else x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * (1 + w.double())


def rotated(x, pos, inv_freq):
    """Half split: element i turns with i + len(inv_freq).  (values, magnitudes that a rounding of cos and sin is relative to)"""
    h = inv_freq.shape[0]
    a = (pos.double()[:, None] * inv_freq.double()[None, :])[:, None, :]
    lo, hi, rest = x[..., :h], x[..., h:2 * h], x[..., 2 * h:]
    size = torch.cat([lo.abs() + hi.abs(), lo.abs() + hi.abs(), rest.abs()], -1)
    return torch.cat([lo * a.cos() - hi * a.sin(), hi * a.cos() + lo * a.sin(), rest], -1), size


def append(c, q_norm, k_norm, eps, inv_freq, positions=None):
    """Expected (q_out, k_cache, v_cache) in 64 bits and how far each value of the first two may be off: one rounding to BF16, a norm whose sum of
    dim squares in FP32 is off by dim * 2^-24 at most (half of that in its root) with six more roundings, cos and sin by 4e-7."""
    out, kc, vc = c.out.double().clone(), c.k_cache.double().clone(), c.v_cache.double().clone()
    q_tol, k_tol = torch.zeros_like(out), torch.zeros_like(kc)
    rel = (c.dim / 2 + 8) * 2.0 ** -24 + 4e-7
    for s, (n, kv) in enumerate(zip(c.new, c.kv)):
        for i in range(n):
            p, t = kv - n + i, int(c.starts[s]) + i
            if p < 0:
                continue
            angle = torch.tensor([p if positions is None else int(positions[t])], device=out.device)
            y, size = rotated(normed(c.q[t:t + 1], q_norm, eps), angle, inv_freq)
            out[t], q_tol[t] = y[0], BF16_HALF_STEP * y[0].abs() + rel * size[0] + 1e-30
            y, size = rotated(normed(c.k[t:t + 1], k_norm, eps), angle, inv_freq)
            page, slot = int(c.table[s, p // c.page]), p % c.page
            c.by_token(kc)[page, slot], c.by_token(k_tol)[page, slot] = y[0], BF16_HALF_STEP * y[0].abs() + rel * size[0] + 1e-30
            c.by_token(vc)[page, slot] = c.v[t].double()
    return (out, q_tol), (kc, k_tol), vc


def worst(got, want, tol):
    """The largest error in units of what is allowed (values that may not change: any change is infinite)."""
    got = got.double()
    off = (got - want).abs()
    off = torch.where(torch.isfinite(got), off, torch.full_like(off, float("inf")))
    return float(torch.where(off == 0, torch.zeros_like(off), off / tol).max()) if off.numel() else 0.0
