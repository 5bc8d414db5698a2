"""The paged K/V cache operators as cases that can be timed and checked: rotary positions, appending to a paged cache,
attention over a cache of 16-bit pages and over one of 4-bit (MXFP4) pages.

A case is a dict of plain values.  `prepare` makes what a program has in hand before the call, `run` is one pass through
an operator: its plain form in elementary torch operations (own = False) or the calls a user makes of libqasr
(own = True).  `exact` computes the same outputs from the definition in 64 bits.

Definitions
  rotary   y = x, or x / sqrt(mean(x^2) + eps) * w over the head where a norm weight is given; then for the pairs (a, b)
           of the first `rot` dims (half layout: dims i and i + rot/2; interleaved: 2i and 2i + 1)
           a' = a cos - b sin, b' = b cos + a sin with the table row of the token's position; the other dims pass.
  append   K rotated as above and V as it is, written to page table[seq][pos // page] at offset pos % page.
  mxfp4    a block of 32 dims holds E, the smallest exponent in [-23, 13] with amax <= 6 * 2^E, and 32 e2m1 codes: the
           values +-{0, .5, 1, 1.5, 2, 3, 4, 6} * 2^E nearest to x (ties to the even code).
  attend   row i of a sequence's n queries sits at position p = kv_len - n + i; its keys are all of the sequence's, or
           those at positions <= p (causal), of these the last `window` (window > 0); o = softmax(scale q.k) v, and
           zeros for a row with no key.

Page layouts (hd = head_dim, one (page, head) block each, pages in a pool [page][kv head]):
  16 bit   [token][hd]
  mxfp4    codes, then scale bytes (E + 127).
           K codes: per token the dims in the order (d % 32) / 8, d / 32, d % 8; two codes a byte, the even dim low.
           K scales: [token][hd / 32].
           V codes: per 16 tokens the order (t % 16) / 4, d / (hd / 16), t % 4, d % (hd / 16).
           V scales: per 16 tokens [hd / 32][16].
"""
import math

import numpy as np
import torch

own = False

DEV = "cuda:0"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
EPS = 1e-6


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # one decode step of one utterance: the 16 query heads of the decoder, fresh from the f32 QKV product, normed
        {"name": "rope step", "op": "rope", "rows": 1, "heads": 16, "hd": 128, "rot": 128, "inter": False, "norm": True,
         "x": "f32", "y": "f16", "ld": 4096, "n_pos": 32768},
        # a packed prompt batch whose heads lie in the wider QKV rows, half of each head rotated in pairs
        {"name": "rope prompt", "op": "rope", "rows": 8192, "heads": 16, "hd": 128, "rot": 64, "inter": True,
         "norm": False, "x": "bf16", "y": "bf16", "ld": 4096, "n_pos": 32768},
        # the table of a model stretched to four times its trained context
        {"name": "rope table", "op": "table", "n_pos": 131072, "rot": 128, "kind": 3, "theta": 1e6, "factor": 4.0,
         "orig": 32768},
        # one decode step of 64 utterances, K and V from the f32 QKV rows
        {"name": "append step", "op": "append", "rows": 64, "n_seq": 64, "kvh": 8, "hd": 128, "rot": 128, "inter": False,
         "norm": True, "x": "f32", "kv": "f16", "page": 16, "max_kv": 1024, "ld": 4096},
        # a packed prompt batch of 21 utterances of odd lengths
        {"name": "append prompt", "op": "append", "rows": 8191, "n_seq": 21, "kvh": 8, "hd": 128, "rot": 128,
         "inter": False, "norm": True, "x": "f32", "kv": "bf16", "page": 64, "max_kv": 1024, "ld": 4096},
        # the same into 4-bit pages, read back as values
        {"name": "append prompt 4-bit", "op": "append", "rows": 8191, "n_seq": 21, "kvh": 8, "hd": 128, "rot": 128,
         "inter": False, "norm": True, "x": "f32", "kv": "mxfp4", "page": 64, "max_kv": 1024, "ld": 4096},
        # one token of one 30 s utterance: where latency counts
        {"name": "decode short", "op": "attend", "n_seq": 1, "n_q": 1, "min_kv": 403, "max_kv": 403, "heads": 16,
         "kvh": 8, "hd": 128, "causal": True, "window": 0, "q": "f16", "kv": "f16", "page": 16},
        # one token of one session at its full context
        {"name": "decode long", "op": "attend", "n_seq": 1, "n_q": 1, "min_kv": 32768, "max_kv": 32768, "heads": 16,
         "kvh": 8, "hd": 128, "causal": True, "window": 0, "q": "f16", "kv": "f16", "page": 64},
        # one token of 64 sessions of very different lengths
        {"name": "decode batch", "op": "attend", "n_seq": 64, "n_q": 1, "min_kv": 17, "max_kv": 8200, "heads": 16,
         "kvh": 8, "hd": 128, "causal": True, "window": 0, "q": "bf16", "kv": "bf16", "page": 16},
        # a long recording's prompt: every row against all before it
        {"name": "prompt", "op": "attend", "n_seq": 2, "n_q": 4097, "min_kv": 6001, "max_kv": 8192, "heads": 16,
         "kvh": 8, "hd": 128, "causal": True, "window": 0, "q": "f16", "kv": "f16", "page": 64},
        # one token of 32 sessions up to the full context, over 4-bit pages
        {"name": "decode batch 4-bit", "op": "attend", "n_seq": 32, "n_q": 1, "min_kv": 501, "max_kv": 32768,
         "heads": 16, "kvh": 8, "hd": 128, "causal": True, "window": 0, "q": "f16", "kv": "mxfp4", "page": 64},
        # a chunk of a prompt on a long 4-bit context
        {"name": "prompt chunk 4-bit", "op": "attend", "n_seq": 3, "n_q": 511, "min_kv": 8000, "max_kv": 16384,
         "heads": 16, "kvh": 8, "hd": 128, "causal": True, "window": 0, "q": "bf16", "kv": "mxfp4", "page": 64},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def draw(rng):
    op = rng.choice(["rope", "table", "append", "append", "attend", "attend", "attend", "attend"])
    hd = rng.choice([64, 128, 128, 256])
    if op == "table":
        return {"op": op, "n_pos": _log(rng, 100, 131072), "rot": rng.choice([32, 64, 80, 128]),
                "kind": rng.choice([0, 1, 2, 3]), "theta": rng.choice([1e4, 1e6]),
                "factor": rng.choice([2.0, 4.0, 8.0]), "orig": rng.choice([4096, 32768])}
    rot = hd // rng.choice([1, 1, 2, 4])
    kvh, g = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 2, 4, 5])
    common = {"hd": hd, "rot": rot, "inter": rng.random() < 0.4, "norm": rng.random() < 0.5,
              "x": rng.choice(["f32", "f32", "f16", "bf16"])}
    if op == "rope":
        rows, heads = _log(rng, 1, 8192), kvh * g
        rows = min(rows, 8192 * 16 * 128 // (heads * hd))
        return {"op": op, "rows": rows, "heads": heads, **common, "y": rng.choice(["f16", "bf16", "f32"]),
                "ld": heads * hd + rng.choice([0, 0, kvh * hd, 8, 3]), "n_pos": 32768}
    if op == "append":
        n_seq = _log(rng, 1, 64)
        rows = max(n_seq, min(_log(rng, 1, 8191), 8191 * 8 * 128 // (kvh * hd)))
        return {"op": op, "rows": rows, "n_seq": n_seq, "kvh": kvh, **common,
                "kv": rng.choice(["f16", "bf16", "mxfp4", "mxfp4"]), "page": rng.choice([16, 32, 64, 128]),
                "max_kv": 128 * (1 + 2 * rows // n_seq // 128), "ld": kvh * hd + rng.choice([0, kvh * hd, 8, 5])}
    kv, q = rng.choice(["f16", "bf16", "mxfp4", "mxfp4"]), rng.choice(["f16", "bf16"])
    case = {"op": op, "heads": kvh * g, "kvh": kvh, "hd": hd, "q": q if kv == "mxfp4" else kv, "kv": kv,
            "page": rng.choice([16, 32, 64, 128]), "causal": rng.random() < 0.8,
            "window": rng.choice([0, 0, 0, 100, 1000])}
    if rng.random() < 0.6:    # single tokens and short verify passes
        n_seq, n_q = _log(rng, 1, 64), rng.choice([1, 1, 1, 2, 7])
        max_kv = _log(rng, 16, min(32768, 500000 // n_seq))
    else:                     # prompts and chunks of them
        n_seq, n_q = rng.choice([1, 2, 3, 5]), _log(rng, 16, 2500)
        max_kv = _log(rng, n_q, 8192)
    return {**case, "n_seq": n_seq, "n_q": n_q, "max_kv": max_kv, "min_kv": _log(rng, 1, max_kv)}


# ------------------------------------------------------------------------------------------------ inputs
def _rand(gen, *shape, scale=1.0):
    return torch.randn(*shape, generator=gen, device=DEV, dtype=torch.float32) * scale


def _lengths(case):
    """Each sequence's keys, spread over the logarithm of the case's range with the longest among them, and its
    queries, some sequences with fewer than the first.  They go by the case alone, so that `work` can count them."""
    lo, hi = case["min_kv"], case["max_kv"]
    r = np.random.RandomState(case["n_seq"] * 7919 + hi)
    kv = np.exp(r.uniform(math.log(lo), math.log(hi + 0.5), case["n_seq"])).astype(np.int64)
    kv = np.clip(kv, lo, hi)
    kv[r.randint(case["n_seq"])] = hi
    nq = np.minimum(kv, case["n_q"])
    nq[1:] -= np.arange(1, len(nq)) * (nq[1:] // 7)
    return kv, np.maximum(nq, 1)


def _pages(case, seed, kv):
    """A page table of each sequence's own pages in no order, as an allocator leaves them; unused entries are -1."""
    page = case["page"]
    per = (kv + page - 1) // page
    width, used = int(max(1, per.max())), int(per.sum())
    n_pages = used + 3
    r = np.random.RandomState((seed + 1) % (1 << 31))
    ids = r.permutation(n_pages)[:used]
    table = np.full((len(kv), width), -1, np.int32)
    table[np.arange(width)[None] < per[:, None]] = ids
    return n_pages, torch.from_numpy(table).to(DEV)


def _table(case, n_pos):
    """cos and sin of every position, [n_pos][rot/2][2], from 64-bit angles."""
    pos = torch.arange(n_pos, device=DEV, dtype=torch.float64)
    f = 1e6 ** (-torch.arange(0, case["rot"], 2, device=DEV, dtype=torch.float64) / case["rot"])
    a = pos[:, None] * f
    return torch.stack((a.cos(), a.sin()), -1).float().contiguous()


def _outlying(gen, *shape):
    """Projections with a few loud channels, as key vectors have."""
    x = _rand(gen, *shape)
    return x * (1 + 4 * (torch.rand(shape[-1], generator=gen, device=DEV) < 0.04))


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(int(seed))
    op = case["op"]
    if op == "table":
        # which stretch of positions: the first one, moved by the seed as a session moves through a recording
        return {"case": case, "first": int(seed) % 1009}
    state = {"case": case}
    if op in ("rope", "append"):
        state["norm_w"] = 1 + 0.1 * _rand(gen, case["hd"]) if case["norm"] else None
    if op == "rope":
        x = _outlying(gen, case["rows"], case["ld"]).to(TYPES[case["x"]])
        state["x"] = x[:, : case["heads"] * case["hd"]]
        state["pos"] = torch.randint(0, case["n_pos"], (case["rows"],), generator=gen, device=DEV, dtype=torch.int32)
        state["cs"] = _table(case, case["n_pos"])
        state["y"] = torch.empty(case["rows"], case["heads"] * case["hd"], device=DEV, dtype=TYPES[case["y"]])
        return state
    if op == "append":
        n, width = case["n_seq"], case["kvh"] * case["hd"]
        r = np.random.RandomState(case["rows"] * 7919 + n)   # lengths go by the case alone
        cut = np.sort(r.choice(np.arange(1, case["rows"]), n - 1, replace=False)) if n > 1 else np.zeros(0, np.int64)
        new = np.diff(np.concatenate([[0], cut, [case["rows"]]]))
        new = np.minimum(new, case["max_kv"])
        had = np.array([r.randint(0, case["max_kv"] - m + 1) for m in new])
        seq = np.repeat(np.arange(n), new)
        pos = np.concatenate([np.arange(h, h + m) for h, m in zip(had, new)])
        state["n_pages"], state["pages"] = _pages(case, seed, had + new)
        rows = state["rows"] = len(seq)
        state["seq"] = torch.from_numpy(seq.astype(np.int32)).to(DEV)
        state["pos"] = torch.from_numpy(pos.astype(np.int32)).to(DEV)
        state["cs"] = _table(case, case["max_kv"])
        state["k"] = _outlying(gen, rows, case["ld"]).to(TYPES[case["x"]])[:, :width]
        state["v"] = _rand(gen, rows, case["ld"]).to(TYPES[case["x"]])[:, :width]
        shape = (state["n_pages"], case["kvh"], case["page"], case["hd"])
        if case["kv"] == "mxfp4":
            size = state["n_pages"] * case["kvh"] * case["page"] * case["hd"] * 17 // 32
            state["pool"] = [torch.zeros(size, device=DEV, dtype=torch.uint8) for _ in range(2)]
            state["out"] = [torch.empty(rows, width, device=DEV) for _ in range(2)]
        else:
            state["pool"] = [_rand(gen, *shape).to(TYPES[case["kv"]]) for _ in range(2)]
        return state
    kv, nq = _lengths(case)
    state["n_pages"], state["pages"] = _pages(case, seed, kv)
    shape = (state["n_pages"], case["kvh"], case["page"], case["hd"])
    state["q_start"] = torch.from_numpy(np.concatenate([[0], np.cumsum(nq)]).astype(np.int32)).to(DEV)
    state["kv_len"] = torch.from_numpy(kv.astype(np.int32)).to(DEV)
    state["max_q"], state["max_kv"], state["rows"] = int(nq.max()), int(kv.max()), int(nq.sum())
    state["scale"] = case["hd"] ** -0.5
    state["q"] = (_rand(gen, state["rows"], case["heads"] * case["hd"], scale=1.3)).to(TYPES[case["q"]])
    k, v = _rand(gen, *shape), _rand(gen, *shape) + 0.3 * _rand(gen, case["hd"])
    if case["kv"] == "mxfp4":
        state["pool"] = [_pack(*_quantise(k), False), _pack(*_quantise(v), True)]
    else:
        state["pool"] = [k.to(TYPES[case["kv"]]), v.to(TYPES[case["kv"]])]
    state["o"] = torch.empty_like(state["q"])
    return state


# ------------------------------------------------------------------------------------------------ plain forms
def _pow2(e):
    """2^e in f32 from its bits, exact"""
    return (e.to(torch.int32) + 127 << 23).view(torch.float32)


def _quantise(x):
    """f32 [..., hd] -> e2m1 codes (uint8) and exponents [..., hd / 32] by the rule above."""
    b = x.unflatten(-1, (-1, 32))
    m, e = torch.frexp(b.abs().amax(-1))              # amax = m 2^e, m in [.5, 1)
    e = (e - torch.where(m <= 0.75, 3, 2)).clamp(-23, 13)
    a = b.abs() * _pow2(-e)[..., None]
    odd = [a > t for t in (0.25, 1.25, 2.5, 5.0)]      # a tie goes down, to the even code
    even = [a >= t for t in (0.75, 1.75, 3.5)]         # a tie goes up, to the even code
    code = sum(t.to(torch.uint8) for t in odd + even)
    return (code + 8 * torch.signbit(b).to(torch.uint8)).flatten(-2), e


def _value(code, e):
    """The f32 values of e2m1 codes [..., hd] and exponents [..., hd / 32]."""
    grid = torch.tensor(GRID + tuple(-g for g in GRID), device=code.device, dtype=torch.float32)
    return (grid[code.long()].unflatten(-1, (-1, 32)) * _pow2(e)[..., None]).flatten(-2)


def _pack(code, e, is_v):
    """Codes [pages][heads][tokens][hd] and exponents into a pool of bytes in the page layout."""
    hd = code.shape[-1]
    s = (e + 127).to(torch.uint8)
    if is_v:
        c = code.unflatten(-1, (16, hd // 16)).unflatten(2, (-1, 4, 4)).permute(0, 1, 2, 3, 5, 4, 6)
        s = s.unflatten(2, (-1, 16)).transpose(-1, -2)
    else:
        c = code.unflatten(-1, (-1, 4, 8)).transpose(-2, -3)
    c = c.reshape(*code.shape[:2], -1, 2)
    return torch.cat((c[..., 0] | c[..., 1] << 4, s.reshape(*code.shape[:2], -1)), -1).flatten()


def _unpack(pool, case, is_v):
    """The inverse: a pool of bytes -> f32 [pages][heads][tokens][hd]."""
    page, hd = case["page"], case["hd"]
    p = pool.view(-1, case["kvh"], page * hd * 17 // 32)
    b, s = p[..., : page * hd // 2], p[..., page * hd // 2:]
    c = torch.stack((b & 15, b >> 4), -1).flatten(-2)
    if is_v:
        c = c.view(*c.shape[:2], page // 16, 4, 16, 4, hd // 16).permute(0, 1, 2, 3, 5, 4, 6)
        s = s.reshape(*s.shape[:2], page // 16, hd // 32, 16).transpose(-1, -2)
    else:
        c = c.view(*c.shape[:2], page, 4, hd // 32, 8).transpose(-2, -3)
    e = s.reshape(*s.shape[:2], page, hd // 32).to(torch.int32) - 127
    return _value(c.reshape(*c.shape[:2], page, hd), e)


def _rotated(x, norm_w, cs, pos, case):
    """Heads [rows][heads][hd], normed and rotated, in x's type (32 or 64 bits)."""
    if norm_w is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * norm_w.to(x.dtype)
    rot = case["rot"]
    t = cs[pos.long()].to(x.dtype)[:, None]
    c, s = t[..., 0], t[..., 1]
    if case["inter"]:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        r = torch.stack((a * c - b * s, b * c + a * s), -1).flatten(-2)
    else:
        a, b = x[..., : rot // 2], x[..., rot // 2: rot]
        r = torch.cat((a * c - b * s, b * c + a * s), -1)
    return torch.cat((r, x[..., rot:]), -1)


def _plain_table(state):
    c = state["case"]
    rot, kind, theta, factor = c["rot"], c["kind"], c["theta"], c["factor"]
    i = torch.arange(0, rot, 2, device=DEV, dtype=torch.float64)
    mscale = 1.0
    if kind == 2:
        theta = theta * factor ** (rot / (rot - 2))
    f = theta ** (-i / rot)
    if kind == 1:
        f = f / factor
    if kind == 3:
        at = lambda beta: rot * math.log(c["orig"] / (beta * 2 * math.pi)) / (2 * math.log(theta))  # noqa: E731
        lo, hi = max(math.floor(at(32.0)), 0), min(math.ceil(at(1.0)), rot - 1)
        ramp = ((i / 2 - lo) / max(hi - lo, 1e-3)).clamp(0, 1)
        f = f * (1 - ramp) + f / factor * ramp
        mscale = 0.1 * math.log(factor) + 1
    a = torch.arange(state["first"], state["first"] + c["n_pos"], device=DEV, dtype=torch.float64)[:, None] * f
    return torch.stack((a.cos() * mscale, a.sin() * mscale), -1).float()


def _plain_append(state):
    case = state["case"]
    k = state["k"].unflatten(-1, (case["kvh"], case["hd"]))
    v = state["v"].unflatten(-1, (case["kvh"], case["hd"])).float()
    # in 64 bits for 4-bit pages: a key next to a border between two codes falls on its own side
    k = k.double() if case["kv"] == "mxfp4" else k.float()
    k = _rotated(k, state["norm_w"], state["cs"], state["pos"], case).float()
    if case["kv"] == "mxfp4":
        return [_value(*_quantise(x)).flatten(-2) for x in (k, v)]
    seq, pos = state["seq"].long(), state["pos"].long()
    page = state["pages"][seq, pos // case["page"]].long()
    pk, pv = state["pool"]
    pk[page, :, pos % case["page"]] = k.to(pk.dtype)
    pv[page, :, pos % case["page"]] = v.to(pv.dtype)
    return [pk, pv]


def _plain_attend(state):
    case = state["case"]
    h, kvh, hd = case["heads"], case["kvh"], case["hd"]
    q_start, kv = state["q_start"].long(), state["kv_len"].long()
    n, nq = case["n_seq"], q_start[1:] - q_start[:-1]
    i = torch.arange(state["max_q"], device=DEV)
    row = (q_start[:-1, None] + i).clamp(max=state["rows"] - 1)
    q = state["q"].float().unflatten(-1, (kvh, h // kvh, hd))[row].permute(0, 2, 1, 3, 4).flatten(2, 3)
    pages = state["pages"].clamp(min=0).long()
    pools = [_unpack(p, case, j == 1) for j, p in enumerate(state["pool"])] if case["kv"] == "mxfp4" else state["pool"]
    k, v = (p[pages].transpose(1, 2).flatten(2, 3)[:, :, : state["max_kv"]].float() for p in pools)
    s = torch.matmul(q, k.transpose(-1, -2)) * state["scale"]
    s = s.view(n, kvh, state["max_q"], h // kvh, -1)
    key, at = torch.arange(k.shape[2], device=DEV), (kv - nq)[:, None] + i
    ok = (key < kv[:, None])[:, None].expand(-1, state["max_q"], -1)
    if case["causal"]:
        ok = ok & (key <= at[..., None])
    if case["window"]:
        ok = ok & (key > at[..., None] - case["window"])
    s = s.masked_fill(~ok[:, None, :, None], -math.inf)
    top = s.amax(-1, keepdim=True).clamp(min=-1e30)
    p = torch.exp(s - top)
    o = torch.matmul(p.flatten(2, 3), v).view(n, kvh, state["max_q"], h // kvh, hd)
    o = o / p.sum(-1, keepdim=True).clamp(min=1e-30)
    o = o.permute(0, 2, 1, 3, 4).flatten(2)
    return o[i < nq[:, None]].to(TYPES[case["q"]])


# ------------------------------------------------------------------------------------------------ one pass
def _plain(state):
    case = state["case"]
    if case["op"] == "table":
        return _plain_table(state)
    if case["op"] == "rope":
        x = state["x"].float().unflatten(-1, (case["heads"], case["hd"]))
        return _rotated(x, state["norm_w"], state["cs"], state["pos"], case).flatten(-2).to(TYPES[case["y"]])
    return _plain_append(state) if case["op"] == "append" else _plain_attend(state)


def _handles(state):
    """What a program keeps between calls: the library, the cache and call descriptions, the workspace."""
    import ctypes
    import os
    import sys

    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "light-whisper_amd")
    if root not in sys.path:
        sys.path.insert(0, root)
    from qasr import _lib

    case, lib = state["case"], _lib.load()
    ids = {"f32": _lib.T_F32, "f16": _lib.T_F16, "bf16": _lib.T_BF16, "mxfp4": _lib.T_MXFP4}
    h = {"lib": lib, "check": _lib.check, "ids": ids, "ref": ctypes.byref}
    if case["op"] == "table":
        h["scaling"] = _lib.RopeScaling(rot_dim=case["rot"], kind=case["kind"], theta=case["theta"],
                                        factor=case["factor"], orig_ctx=case["orig"], beta_fast=32.0, beta_slow=1.0)
        h["out"] = torch.empty(case["n_pos"], case["rot"] // 2, 2, device=DEV)
    if case["op"] in ("rope", "append"):
        w = state["norm_w"]
        h["rope"] = _lib.Rope(cs=state["cs"].data_ptr(), n_pos=state["cs"].shape[0], rot_dim=case["rot"],
                              interleaved=int(case["inter"]), norm_w=w.data_ptr() if w is not None else None, eps=EPS)
    if case["op"] in ("append", "attend"):
        h["cache"] = _lib.KvCache(k=state["pool"][0].data_ptr(), v=state["pool"][1].data_ptr(),
                                  page_table=state["pages"].data_ptr(), n_seq=case["n_seq"],
                                  max_pages=state["pages"].shape[1], n_pages=state["n_pages"], page_size=case["page"],
                                  n_kv_heads=case["kvh"], head_dim=case["hd"], type=ids[case["kv"]])
    if case["op"] == "attend":
        h["attn"] = _lib.PagedAttn(n_heads=case["heads"], q_type=ids[case["q"]], o_type=ids[case["q"]],
                                   causal=int(case["causal"]), window=case["window"], scale=state["scale"],
                                   max_q=state["max_q"], max_kv=state["max_kv"])
        size = ctypes.c_size_t()
        _lib.check(lib.qasr_paged_attention_workspace(ctypes.byref(h["cache"]), ctypes.byref(h["attn"]),
                                                      ctypes.byref(size)))
        h["ws"] = torch.zeros(max(1, size.value), device=DEV, dtype=torch.uint8)
        h["ws_bytes"] = size.value
    return h


def _own(state):
    h = state.get("handles")
    if h is None:
        h = state["handles"] = _handles(state)
    case, lib, check, ref, ids = state["case"], h["lib"], h["check"], h["ref"], h["ids"]
    stream = torch.cuda.current_stream().cuda_stream
    if case["op"] == "table":
        check(lib.qasr_op_rope_table_scaled(ref(h["scaling"]), state["first"], case["n_pos"], h["out"].data_ptr(),
                                            stream))
        return h["out"]
    if case["op"] == "rope":
        x, y = state["x"], state["y"]
        check(lib.qasr_op_rope(x.data_ptr(), ids[case["x"]], case["ld"], state["pos"].data_ptr(), case["rows"],
                               case["heads"], case["hd"], ref(h["rope"]), y.data_ptr(), ids[case["y"]], y.shape[1],
                               stream))
        return y
    if case["op"] == "append":
        seq, pos, rows = state["seq"].data_ptr(), state["pos"].data_ptr(), state["rows"]
        check(lib.qasr_op_kv_append(ref(h["cache"]), state["k"].data_ptr(), state["v"].data_ptr(), ids[case["x"]],
                                    case["ld"], case["ld"], seq, pos, rows, ref(h["rope"]), stream))
        if case["kv"] != "mxfp4":
            return state["pool"]
        k, v = state["out"]
        check(lib.qasr_op_kv_gather(ref(h["cache"]), seq, pos, rows, k.data_ptr(), v.data_ptr(), ids["f32"],
                                    k.shape[1], v.shape[1], stream))
        return [k, v]
    q, o = state["q"], state["o"]
    check(lib.qasr_op_paged_attention(ref(h["cache"]), ref(h["attn"]), q.data_ptr(), q.shape[1],
                                      state["q_start"].data_ptr(), state["kv_len"].data_ptr(), state["rows"],
                                      o.data_ptr(), o.shape[1], h["ws"].data_ptr(), h["ws_bytes"], stream))
    return o


def run(state):
    return _own(state) if own else _plain(state)


# ------------------------------------------------------------------------------------------------ what a pass needs
_SIZE = {"f32": 4.0, "f16": 2.0, "bf16": 2.0, "mxfp4": 17.0 / 32.0}


def work(case):
    op = case["op"]
    if op == "table":
        return {"bytes": 4 * case["n_pos"] * case["rot"], "flops": 4 * case["n_pos"] * case["rot"]}
    if op == "rope":
        n = case["rows"] * case["heads"] * case["hd"]
        table = 4 * case["rot"] * min(case["rows"], case["n_pos"])
        return {"bytes": n * (_SIZE[case["x"]] + _SIZE[case["y"]]) + table, "flops": 6 * n}
    if op == "append":
        n = 2 * case["rows"] * case["kvh"] * case["hd"]
        out = _SIZE[case["kv"]] + (_SIZE["mxfp4"] + 4 if case["kv"] == "mxfp4" else 0)
        return {"bytes": n * (_SIZE[case["x"]] + out) + 4 * case["rot"] * min(case["rows"], case["max_kv"]),
                "flops": 6 * n}
    kv, nq = _lengths(case)
    keys = kv * nq - (nq * (nq - 1) // 2 if case["causal"] else 0)
    seen = kv
    if case["window"]:
        keys = np.minimum(keys, nq * case["window"])
        seen = np.minimum(kv, nq + case["window"])
    return {"bytes": float(2 * seen.sum() * case["kvh"] * case["hd"] * _SIZE[case["kv"]]
                           + 2 * nq.sum() * case["heads"] * case["hd"] * _SIZE[case["q"]]),
            "flops": float(4 * keys.sum() * case["heads"] * case["hd"])}


# ------------------------------------------------------------------------------------------------ in 64 bits
def _exact_rope(x, w, cs, pos, case):
    """numpy, [rows][heads][hd] float64"""
    if w is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + EPS) * w
    rot, y = case["rot"], x.copy()
    z = cs[pos, :, 0][:, None] + 1j * cs[pos, :, 1][:, None]
    first, second = (slice(0, rot, 2), slice(1, rot, 2)) if case["inter"] else (slice(0, rot // 2), slice(rot // 2, rot))
    r = (x[..., first] + 1j * x[..., second]) * z
    y[..., first], y[..., second] = r.real, r.imag
    return y


def _exact_fp4(x):
    """numpy float64 [..., hd] -> the nearest representable values"""
    b = x.reshape(*x.shape[:-1], -1, 32)
    amax = np.abs(b).max(-1, keepdims=True)
    with np.errstate(divide="ignore"):
        e = np.ceil(np.log2(amax / 6.0))
    e = np.where(6.0 * np.exp2(e - 1) >= amax, e - 1, np.where(6.0 * np.exp2(e) < amax, e + 1, e))
    e = np.clip(np.where(amax > 0, e, -23), -23, 13)
    a = np.abs(b) / np.exp2(e)
    step = np.where(a < 2, 0.5, np.where(a < 4, 1.0, 2.0))   # the grid is even in each of these stretches
    a = np.minimum(np.rint(a / step) * step, 6.0)            # rint: ties to even, which is the even code
    return (np.copysign(a, b) * np.exp2(e)).reshape(x.shape)


def exact(case, seed):
    op = case["op"]
    state = prepare(case, seed)
    num = lambda t: t.double().cpu().numpy()  # noqa: E731
    if op == "table":
        rot, theta, factor = case["rot"], case["theta"], case["factor"]
        if case["kind"] == 2:
            theta *= factor ** (rot / (rot - 2))
        f, m = np.array([theta ** (-2.0 * j / rot) for j in range(rot // 2)]), 1.0
        if case["kind"] == 1:
            f = f / factor
        if case["kind"] == 3:
            dim = lambda turns: rot / 2 * math.log(case["orig"] / (2 * math.pi * turns), theta)  # noqa: E731
            lo, hi = max(math.floor(dim(32)), 0), min(math.ceil(dim(1)), rot - 1)
            keep = 1 - np.clip((np.arange(rot // 2) - lo) / max(hi - lo, 1e-3), 0, 1)
            f, m = f * keep + f / factor * (1 - keep), 0.1 * math.log(factor) + 1
        a = np.outer(np.arange(state["first"], state["first"] + case["n_pos"], dtype=np.float64), f)
        return m * np.stack((np.cos(a), np.sin(a)), -1)
    if op in ("rope", "append"):
        w = num(state["norm_w"]) if state["norm_w"] is not None else None
        cs, pos = num(state["cs"]), state["pos"].cpu().numpy()
    if op == "rope":
        x = num(state["x"]).reshape(-1, case["heads"], case["hd"])
        return _exact_rope(x, w, cs, pos, case).reshape(x.shape[0], -1)
    if op == "append":
        k, v = (num(state[n]).reshape(-1, case["kvh"], case["hd"]) for n in ("k", "v"))
        k = _exact_rope(k, w, cs, pos, case)
        if case["kv"] == "mxfp4":
            # the codes are those of the value rounded to 32 bits, as the definition's input is
            return [_exact_fp4(x.astype(np.float32).astype(np.float64)).reshape(len(x), -1) for x in (k, v)]
        table, seq, out = state["pages"].cpu().numpy(), state["seq"].cpu().numpy(), []
        for pool, x in zip(state["pool"], (k, v)):
            p = num(pool)
            p[table[seq, pos // case["page"]], :, pos % case["page"]] = x
            out.append(p)
        return out
    cpu = [t.cpu().numpy() for t in (state["q_start"], state["kv_len"])]
    pools = [_unpack(p, case, j == 1) for j, p in enumerate(state["pool"])] if case["kv"] == "mxfp4" else state["pool"]
    g, hd = case["heads"] // case["kvh"], case["hd"]
    out = torch.zeros(state["rows"], case["heads"], hd, dtype=torch.float64, device=DEV)
    q = state["q"].double().view(-1, case["heads"], hd)
    for s in range(case["n_seq"]):
        r0, r1, n = int(cpu[0][s]), int(cpu[0][s + 1]), int(cpu[1][s])
        ids = state["pages"][s, : (n + case["page"] - 1) // case["page"]].long()
        for h in range(case["kvh"]):
            k, v = (p[ids, h].double().reshape(-1, hd)[:n] for p in pools)
            for c in range(r0, r1, 2048):
                d = min(r1, c + 2048)
                at = torch.arange(c, d, device=DEV) - r1 + n
                key = torch.arange(n, device=DEV)
                ok = torch.ones(d - c, n, dtype=torch.bool, device=DEV)
                if case["causal"]:
                    ok &= key[None] <= at[:, None]
                if case["window"]:
                    ok &= key[None] > at[:, None] - case["window"]
                for j in range(h * g, h * g + g):
                    x = torch.where(ok, q[c:d, j] @ k.T * state["scale"], -math.inf)
                    p = torch.exp(x - x.amax(-1, keepdim=True).clamp(min=-1e300))
                    total = p.sum(-1, keepdim=True)
                    out[c:d, j] = torch.where(total > 0, p @ v / total.clamp(min=1e-300), 0.0)
    return out.view(state["rows"], -1)
