"""Performance cases of what stands between the qkv and the output projection of a decoder layer, over a paged cache of keys and values:

  append   queries and keys normed for each head and rotated by their position, keys and values written to their places in the cache;
  attend   causal attention of each sequence's new tokens over its pages: one token (decode), a few (drafted tokens to verify), many (a prompt or a
           chunk of one), or a batch that mixes them; where "gate" is set, the result is multiplied by sigmoid(gate).

Head layouts: the repository's attention block (24 query heads over 2 key-value heads of 256, a quarter of a head rotated) and generic ones.  Sequences'
lengths are spread over their logarithms by the case's own "shape" number, the same for every seed; pages lie in the cache in an order of the seed.
Keys are normed, so they have unit variance; queries are twice as large, which gives scores a deviation of two and rows of attention that favour some keys.
"""
import math
import os
import random
import sys

import torch

own = False

EPS = 1e-6
BF16 = torch.bfloat16


def listed():
    block = {"q_heads": 24, "kv_heads": 2, "dim": 256, "rot": 64, "norm": True}
    wide = {"q_heads": 32, "kv_heads": 8, "dim": 128, "rot": 128, "norm": True}
    plain = {"q_heads": 32, "kv_heads": 8, "dim": 128, "rot": 128, "norm": False}
    return [
        # The append of one decode step of one sequence: the smallest call, all latency.
        {"name": "append_1", "kind": "append", "seqs": 1, "q_lo": 1, "q_hi": 1, "ctx_lo": 777, "ctx_hi": 777, "singles": 0, "page": 16, "gate": True, "pad": 0, "shape": 1, **block},
        # One decode step of a batch padded to the 96 rows that a captured graph was made for, heads without norms.
        {"name": "append_83", "kind": "append", "seqs": 83, "q_lo": 1, "q_hi": 1, "ctx_lo": 16, "ctx_hi": 4096, "singles": 0, "page": 16, "gate": False, "pad": 13, "shape": 2, **plain},
        # Prompts of one prefill step, some of them continued.
        {"name": "append_prompts", "kind": "append", "seqs": 9, "q_lo": 300, "q_hi": 2048, "ctx_lo": 0, "ctx_hi": 2000, "singles": 0, "page": 64, "gate": True, "pad": 0, "shape": 3, **block},
        # Decode of one sequence with a short past.
        {"name": "decode_1", "kind": "attend", "seqs": 1, "q_lo": 1, "q_hi": 1, "ctx_lo": 1500, "ctx_hi": 1500, "singles": 0, "page": 16, "gate": True, "pad": 0, "shape": 4, **block},
        # Decode of one sequence with a long past.
        {"name": "decode_1_long", "kind": "attend", "seqs": 1, "q_lo": 1, "q_hi": 1, "ctx_lo": 131001, "ctx_hi": 131001, "singles": 0, "page": 64, "gate": True, "pad": 0, "shape": 5, **block},
        # Decode of a batch whose sequences are at very different lengths.
        {"name": "decode_64", "kind": "attend", "seqs": 64, "q_lo": 1, "q_hi": 1, "ctx_lo": 128, "ctx_hi": 16384, "singles": 0, "page": 16, "gate": True, "pad": 0, "shape": 6, **block},
        # Decode of a large batch with heads of 128, padded rows behind it.
        {"name": "decode_243", "kind": "attend", "seqs": 243, "q_lo": 1, "q_hi": 1, "ctx_lo": 64, "ctx_hi": 2048, "singles": 0, "page": 32, "gate": False, "pad": 13, "shape": 7, **wide},
        # Three drafted tokens and the one in front of them, verified for a small batch.
        {"name": "verify_12x4", "kind": "attend", "seqs": 12, "q_lo": 4, "q_hi": 4, "ctx_lo": 500, "ctx_hi": 8192, "singles": 0, "page": 16, "gate": True, "pad": 0, "shape": 8, **block},
        # A prompt of odd length.
        {"name": "prefill_149", "kind": "attend", "seqs": 1, "q_lo": 149, "q_hi": 149, "ctx_lo": 0, "ctx_hi": 0, "singles": 0, "page": 16, "gate": True, "pad": 0, "shape": 9, **block},
        # One chunk of 256 tokens, the engine's, far into a long prompt.
        {"name": "prefill_chunk", "kind": "attend", "seqs": 1, "q_lo": 256, "q_hi": 256, "ctx_lo": 16384, "ctx_hi": 16384, "singles": 0, "page": 64, "gate": True, "pad": 0, "shape": 10, **block},
        # A long prompt in one piece, the largest work.
        {"name": "prefill_8192", "kind": "attend", "seqs": 1, "q_lo": 8192, "q_hi": 8192, "ctx_lo": 0, "ctx_hi": 0, "singles": 0, "page": 64, "gate": True, "pad": 0, "shape": 11, **block},
        # A step that mixes prompts of different lengths, some continued, with sequences that decode; heads of 128.
        {"name": "mixed", "kind": "attend", "seqs": 5, "q_lo": 200, "q_hi": 1900, "ctx_lo": 0, "ctx_hi": 2000, "singles": 19, "page": 16, "gate": False, "pad": 5, "shape": 12, **wide},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi))))) if hi > lo else lo


def _lens(case):
    """New tokens and tokens in front of them, for each sequence: those with q_lo..q_hi new ones, then those with a single one."""
    rng = random.Random(case["shape"])
    new = [_log_int(rng, case["q_lo"], case["q_hi"]) for _ in range(case["seqs"])] + [1] * case["singles"]
    past = [_log_int(rng, case["ctx_lo"] + 1, case["ctx_hi"] + 1) - 1 for _ in new]
    return new, past


def _seen(case):
    return sum(n * p + n * (n + 1) // 2 for n, p in zip(*_lens(case)))


def draw(rng):
    """A case of the same ranges: 1 to 256 sequences, 1 to 8192 new tokens, up to 131072 tokens of past, heads of 64, 128 and 256, 1 to 16 query heads for
    a key-value head, pages of 1 to 256 tokens; as large as the largest listed one at most."""
    while True:
        dim = rng.choice([64, 128, 128, 256, 256])
        kv_heads = rng.choice([1, 2, 4, 8])
        group = rng.choice([1, 2, 3, 4, 5, 6, 7, 8, 12, 16])
        case = {"kind": rng.choice(["append", "attend", "attend", "attend"]), "q_heads": kv_heads * group, "kv_heads": kv_heads, "dim": dim,
                "rot": rng.choice([dim, dim // 4, dim // 2]), "norm": rng.random() < 0.7, "gate": rng.random() < 0.5,
                "page": rng.choice([16, 16, 32, 64, 64, 128, 256, 1, 24, 40]), "pad": rng.choice([0, 0, rng.randint(1, 40)]), "shape": rng.randint(100, 1 << 30), "singles": 0}
        if case["q_heads"] > 64:
            continue
        how = rng.choice(["decode", "decode", "verify", "prompt", "chunk", "mixed"])
        if how in ("decode", "verify"):
            case["seqs"] = _log_int(rng, 1, 256)
            q = 1 if how == "decode" else rng.randint(2, 8)
            lo = _log_int(rng, 1, 4000)
            case.update(q_lo=1 if how == "decode" else rng.randint(1, q), q_hi=q, ctx_lo=lo, ctx_hi=_log_int(rng, lo, 131072))
        elif how == "prompt":
            hi = _log_int(rng, 20, 8192)
            case.update(seqs=rng.randint(1, 9), q_lo=_log_int(rng, 9, hi) if hi > 9 else 9, q_hi=hi, ctx_lo=0, ctx_hi=0)
        else:
            hi = _log_int(rng, 32, 2048)
            case.update(seqs=rng.randint(1, 6), q_lo=_log_int(rng, 9, hi), q_hi=hi, ctx_lo=rng.randint(0, 500), ctx_hi=_log_int(rng, 600, 32768))
            if how == "mixed":
                case["singles"] = rng.randint(1, 40)
        new, past = _lens(case)
        tokens, longest = sum(new), max(n + p for n, p in zip(new, past))
        per_token = case["kv_heads"] * dim
        if tokens > 12000 or sum(n + p for n, p in zip(new, past)) * per_token * 4 > 2 << 30:
            continue
        # the plain form works on sequences padded to the longest one
        if case["kind"] == "attend" and (len(new) * max(new) * longest * case["q_heads"] > 24 * 8192 * 8192 or len(new) * longest * per_token > 1 << 30
                                         or _seen(case) * case["q_heads"] * dim > 8192 * 4096 * 24 * 256):
            continue
        return case


# ---------------------------------------------------------------- inputs

class _State:
    pass


_kept = {}


def _library():
    """The package and the handle that a program keeps for the device."""
    if not _kept:
        sys.path.insert(0, os.path.join(os.getcwd(), "qwen3-27b-thor-runner_b200"))
        import nvfp4
        _kept["nvfp4"], _kept["handle"] = nvfp4, nvfp4.Handle(torch.cuda.current_device(), 16 << 20)
    return _kept["nvfp4"], _kept["handle"]


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, device="cuda", generator=gen, dtype=BF16)

    s = _State()
    s.case = c = dict(case)
    s.new, past = _lens(c)
    seqs, dim, hq, hk, page = len(s.new), c["dim"], c["q_heads"], c["kv_heads"], c["page"]
    s.tokens, s.rows = sum(s.new), sum(s.new) + c["pad"]
    s.longest = max(n + p for n, p in zip(s.new, past))
    starts = [0]
    for n in s.new:
        starts.append(starts[-1] + n)
    s.cu_q, s.kv_len = _ints(starts), _ints([n + p for n, p in zip(s.new, past)])
    pages = [(n + p + page - 1) // page for n, p in zip(s.new, past)]
    order = torch.randperm(sum(pages) + 3, device="cuda", generator=gen).to(torch.int32)
    s.table = torch.zeros((seqs, max(pages)), dtype=torch.int32, device="cuda")      # entries behind a sequence's last page name page 0, as engines leave them
    held = torch.arange(max(pages), device="cuda")[None, :] < _ints(pages)[:, None]
    s.table[held] = order[:sum(pages)]
    s.k_cache, s.v_cache = normal(sum(pages) + 3, page, hk, dim), normal(sum(pages) + 3, page, hk, dim)
    # q, gate, k and v as the merged projection leaves them: where there is a gate, it follows q head by head
    wide = 2 if c["gate"] else 1
    qkv = normal(s.rows, (wide * hq + 2 * hk) * dim)
    qg = qkv[:, :wide * hq * dim].view(s.rows, hq, wide * dim)
    s.q, s.gate = qg[..., :dim], qg[..., dim:] if c["gate"] else None
    s.k = qkv[:, wide * hq * dim:(wide * hq + hk) * dim].view(s.rows, hk, dim)
    s.v = qkv[:, (wide * hq + hk) * dim:].view(s.rows, hk, dim)
    s.out = torch.zeros((s.rows, hq, dim), dtype=BF16, device="cuda")
    if c["kind"] == "append":
        qkv.mul_(2.0)
        s.q_norm, s.k_norm = (0.1 * normal(dim), 0.1 * normal(dim)) if c["norm"] else (None, None)
        s.inv_freq = (1e7 ** (-torch.arange(0, c["rot"], 2, dtype=torch.float64) / c["rot"])).to(torch.float32).cuda()
    else:
        s.q = normal(s.rows, hq, dim).mul_(2.0)          # what the append has normed and rotated
    if own:
        nvfp4, s.handle = _library()
        s.cache = nvfp4.KvCache(s.k_cache, s.v_cache)
        s.batch = nvfp4.PagedBatch(s.kv_len, s.table, tokens=s.rows, cu_q=s.cu_q, max_q_len=max(s.new))
    return s


# ---------------------------------------------------------------- one pass

def _places(s):
    """For each token that belongs to a sequence: its sequence, its place among the sequence's new tokens, its position."""
    starts, t = s.cu_q.long(), torch.arange(s.tokens, device="cuda")
    seq = torch.searchsorted(starts, t, right=True) - 1
    at = t - starts[seq]
    return seq, at, s.kv_len.long()[seq] - (starts[seq + 1] - starts[seq]) + at


def _normed(x, w):
    x = x.float()
    return x if w is None else x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * (1.0 + w.float())


def _rotated(x, angle, rot):
    cos, sin = angle.cos().float()[:, None, :], angle.sin().float()[:, None, :]
    a, b = x[..., :rot // 2], x[..., rot // 2:rot]
    return torch.cat([a * cos - b * sin, b * cos + a * sin, x[..., rot:]], -1)


def _append_plain(s):
    c, n = s.case, s.tokens
    seq, _, pos = _places(s)
    angle = pos.double()[:, None] * s.inv_freq.double()[None, :]
    q = _rotated(_normed(s.q[:n], s.q_norm), angle, c["rot"]).to(BF16)
    k = _rotated(_normed(s.k[:n], s.k_norm), angle, c["rot"]).to(BF16)
    page, slot = s.table.long()[seq, pos // c["page"]], pos % c["page"]
    s.k_cache[page, slot] = k
    s.v_cache[page, slot] = s.v[:n]
    s.out[:n] = q
    return {"q": s.out, "k_cache": s.k_cache, "v_cache": s.v_cache}


def _attend_plain(s):
    c, seqs = s.case, len(s.new)
    hq, hk, dim, most = c["q_heads"], c["kv_heads"], c["dim"], max(s.new)
    seq, at, pos = _places(s)
    q = torch.zeros((seqs, most, hq, dim), device="cuda")
    q[seq, at] = s.q[:s.tokens].float()
    last = torch.full((seqs, most), -1, device="cuda")           # the last key that a row sees; rows that are no token see none
    last[seq, at] = pos
    length = s.table.shape[1] * c["page"]
    k = s.k_cache[s.table.long()].reshape(seqs, length, hk, dim)[:, :s.longest].float()
    v = s.v_cache[s.table.long()].reshape(seqs, length, hk, dim)[:, :s.longest].float()
    q = q.view(seqs, most, hk, hq // hk, dim).permute(0, 2, 1, 3, 4).reshape(seqs, hk, -1, dim)
    scores = torch.matmul(q, k.permute(0, 2, 3, 1)).mul_(dim ** -0.5)
    hidden = torch.arange(s.longest, device="cuda")[None, None, :] > last[:, :, None]
    scores.view(seqs, hk, most, hq // hk, s.longest).masked_fill_(hidden[:, None, :, None, :], -math.inf)
    top = scores.amax(-1, keepdim=True).clamp_(min=-1e30)
    p = scores.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p, v.permute(0, 2, 1, 3)) / total.clamp_(min=1e-30)
    o = o.view(seqs, hk, most, hq // hk, dim).permute(0, 2, 1, 3, 4).reshape(seqs, most, hq, dim)[seq, at]
    if s.gate is not None:
        o = o / (1.0 + torch.exp(-s.gate[:s.tokens].float()))
    s.out[:s.tokens] = o.to(BF16)
    return s.out


def run(s):
    c = s.case
    if not own:
        return _append_plain(s) if c["kind"] == "append" else _attend_plain(s)
    if c["kind"] == "append":
        s.handle.kv_append(s.cache, s.batch, s.q, s.k, s.v, s.out, q_norm=s.q_norm, k_norm=s.k_norm, norm_eps=EPS, inv_freq=s.inv_freq)
        return {"q": s.out, "k_cache": s.k_cache, "v_cache": s.v_cache}
    s.handle.paged_attention(s.cache, s.batch, s.q, s.out, gate=s.gate)
    return s.out


def work(case):
    """Bytes: queries, keys and values of the new tokens in and out, or every key and value that is seen once in, queries (and gates) in, the result out;
    with each sequence's row of the page table.  Flops: two products for every key that a query sees."""
    c = case
    new, past = _lens(c)
    tokens, dim = sum(new), c["dim"]
    table = sum(4 * ((n + p + c["page"] - 1) // c["page"]) for n, p in zip(new, past))
    if c["kind"] == "append":
        return {"bytes": 4 * tokens * (c["q_heads"] + 2 * c["kv_heads"]) * dim + 12 * len(new), "flops": 8 * tokens * (c["q_heads"] + c["kv_heads"]) * dim}
    cached = sum(n + p for n, p in zip(new, past))
    return {"bytes": 4 * cached * c["kv_heads"] * dim + (6 if c["gate"] else 4) * tokens * c["q_heads"] * dim + table,
            "flops": 4 * _seen(c) * c["q_heads"] * dim}


# ---------------------------------------------------------------- the definition in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    c = s.case
    hq, hk, dim, page = c["q_heads"], c["kv_heads"], c["dim"], c["page"]
    starts, lens, table = s.cu_q.tolist(), s.kv_len.tolist(), s.table.long()
    if c["kind"] == "append":
        out = {"q": s.out.double(), "k_cache": s.k_cache.double(), "v_cache": s.v_cache.double()}
        freq, half = s.inv_freq.double(), c["rot"] // 2
        for b, n in enumerate(s.new):
            t0 = starts[b]
            pos = torch.arange(lens[b] - n, lens[b], device="cuda")
            turn = torch.polar(torch.ones((n, 1, half), dtype=torch.float64, device="cuda"), (pos.double()[:, None] * freq)[:, None, :])
            done = []
            for x, w in ((s.q, s.q_norm), (s.k, s.k_norm)):
                y = x[t0:t0 + n].double()
                if w is not None:
                    y = y / torch.sqrt(y.pow(2).sum(-1, keepdim=True) / dim + EPS) * (w.double() + 1)
                z = torch.complex(y[..., :half].contiguous(), y[..., half:2 * half].contiguous()) * turn
                done.append(torch.cat([z.real, z.imag, y[..., 2 * half:]], -1))
            out["q"][t0:t0 + n] = done[0]
            out["k_cache"][table[b, pos // page], pos % page] = done[1]
            out["v_cache"][table[b, pos // page], pos % page] = s.v[t0:t0 + n].double()
        return out
    out = s.out.double()
    for b, n in enumerate(s.new):
        rows = slice(starts[b], starts[b] + n)
        where = table[b, :(lens[b] + page - 1) // page]
        k = s.k_cache[where].flatten(0, 1)[:lens[b]].double()
        v = s.v_cache[where].flatten(0, 1)[:lens[b]].double()
        sees = torch.ones((n, lens[b]), dtype=torch.bool, device="cuda").tril(lens[b] - n)
        for h in range(hq):
            scores = s.q[rows, h].double() @ k[:, h // (hq // hk)].T / math.sqrt(dim)
            weights = torch.softmax(torch.where(sees, scores, -math.inf), -1)
            out[rows, h] = weights @ v[:, h // (hq // hk)]
        if s.gate is not None:
            out[rows] *= torch.sigmoid(s.gate[rows].double())
    return out
