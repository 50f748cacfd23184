"""The operators around the INT4 linears of a decoder layer, as measured cases.

A decoder layer on AWQ weights needs, beside its fused linears: the RMS norm with the residual's addition, the rotary
embedding with the append of the new keys and values to a paged cache, the attention of one new token per sequence over
that cache, and the attention of prompts (or chunks of prompts) over it, causal and with an optional sliding window
whose first tokens (sinks) stay visible.

``own`` chooses between the plain forms (elementary torch operations in 32 bits) and the package's entry points.
Sequence lengths belong to a case (they follow from its numbers alone); all values come from the seed.
"""

import random

import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
F8 = torch.float8_e4m3fn
F8_MAX = 448.0
EPS = 1e-5


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # the norm before a layer's qkv at one token: a launch's latency
        dict(name="norm 1x4096 f16", op="norm", rows=1, d=4096, dtype="f16", residual=True, fp8=False),
        # a long prompt's rows with the row count off every tile, quantised for an 8-bit product (lm_head)
        dict(name="norm 4099x8192 bf16 fp8", op="norm", rows=4099, d=8192, dtype="bf16", residual=True, fp8=True),
        # one new token of each of 64 sequences
        dict(name="rope 64 tokens f16", op="rope", batch=64, new=1, max_len=2048, lens=3, hq=32, hkv=32, d=128,
             page=16, dtype="f16"),
        # a batch of prompts, some in chunks behind what is cached already
        dict(name="rope prompts bf16", op="rope", batch=9, new=2048, max_len=4096, lens=5, hq=28, hkv=4, d=128,
             page=16, dtype="bf16"),
        # a chat's next token: one sequence, 1000 tokens in the cache
        dict(name="decode 1x1000 f16", op="decode", batch=1, max_len=1000, lens=0, hq=32, hkv=32, d=128, page=16,
             window=0, sinks=0, dtype="f16"),
        # a serving batch with lengths of all sizes, one slot of it empty
        dict(name="decode 64 ragged bf16", op="decode", batch=64, max_len=8000, lens=7, hq=28, hkv=4, d=128, page=16,
             window=0, sinks=0, dtype="bf16"),
        # one long document: the cache's length is all there is to split
        dict(name="decode 1x131072 bf16", op="decode", batch=1, max_len=131072, lens=0, hq=64, hkv=8, d=128, page=64,
             window=0, sinks=0, dtype="bf16"),
        # streaming: a window of 4096 and the first 4 tokens of long sequences
        dict(name="decode 32 window f16", op="decode", batch=32, max_len=16384, lens=9, hq=32, hkv=8, d=128, page=32,
             window=4096, sinks=4, dtype="f16"),
        # a short question, small heads: latency
        dict(name="prefill 77 f16 d64", op="prefill", batch=1, new=77, max_len=77, lens=0, hq=14, hkv=2, d=64, page=16,
             window=0, sinks=0, dtype="f16"),
        # one long prompt
        dict(name="prefill 8192 f16", op="prefill", batch=1, new=8192, max_len=8192, lens=0, hq=32, hkv=8, d=128,
             page=16, window=0, sinks=0, dtype="f16"),
        # prompts of all lengths in one batch, some behind cached prefixes
        dict(name="prefill ragged bf16", op="prefill", batch=7, new=2048, max_len=2900, lens=11, hq=28, hkv=4, d=128,
             page=16, window=0, sinks=0, dtype="bf16"),
        # a chunk of a long document under a window with sinks
        dict(name="prefill window bf16", op="prefill", batch=1, new=2048, max_len=16000, lens=0, hq=64, hkv=8, d=128,
             page=64, window=4096, sinks=4, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm."""
    return max(lo, min(hi, int(lo * (hi / lo) ** rng.random() + 0.5)))


HEADS = [(32, 32), (32, 8), (28, 4), (64, 8), (40, 40), (14, 2), (16, 1), (12, 12), (40, 8), (20, 4)]


def draw(rng):
    op = rng.choice(["norm", "rope", "decode", "decode", "prefill", "prefill"])
    dtype = rng.choice(["f16", "bf16"])
    if op == "norm":
        d = _log(rng, 128, 16384)
        d = d if rng.random() < 0.25 else d // 8 * 8
        d += 8 * (d == 3072)
        rows = _log(rng, 1, max(1, 4099 * 8192 // d))
        return dict(op=op, rows=rows, d=d, dtype=rng.choice([dtype, dtype, "f32"]), residual=rng.random() < 0.7,
                    fp8=rng.random() < 0.4)
    hq, hkv = rng.choice(HEADS)
    d = rng.choice([64, 128, 128])
    page = rng.choice([8, 16, 16, 24, 32, 64, 128, 256])
    lens = rng.randrange(1, 1 << 20)
    if op == "rope":
        batch = _log(rng, 1, 64)
        new = _log(rng, 1, max(1, 16384 // batch))
        return dict(op=op, batch=batch, new=new, max_len=new + _log(rng, 1, 2048), lens=lens, hq=hq, hkv=hkv, d=d,
                    page=page, dtype=dtype)
    window = rng.choice([0, 0, _log(rng, 16, 8192)])
    sinks = rng.choice([0, 4, rng.randrange(1, 200)]) if window else 0
    if op == "decode":
        batch = _log(rng, 1, 256)
        top = (1 << 20) // (batch * hkv)  # tokens a sequence: the cache stays within the largest listed one
        max_len = _log(rng, 1, max(1, min(131072, top)))
        return dict(op=op, batch=batch, max_len=max_len, lens=rng.choice([0, lens]), hq=hq, hkv=hkv, d=d, page=page,
                    window=window, sinks=sinks, dtype=dtype)
    batch = _log(rng, 1, 16)
    new = _log(rng, 1, 6000 // batch + 1)
    # scores of the padded batch: no more than the longest listed prompt has
    most = (8192 * 8192 * 32) // (2 * batch * hq * new)
    max_len = new + (_log(rng, 1, max(1, min(20000 // batch, most - new))) if rng.random() < 0.6 else 0)
    return dict(op=op, batch=batch, new=new, max_len=max_len, lens=rng.choice([0, lens]), hq=hq, hkv=hkv, d=d,
                page=page, window=window, sinks=sinks, dtype=dtype)


def lengths(case):
    """(new tokens, tokens in the cache with them) of each sequence: all at their largest where "lens" is 0; else the
    first one so, the others spread over their logarithm, and of eight or more the last one an empty slot."""
    b, top, new = case["batch"], case["max_len"], case.get("new", 1)
    r = random.Random(case["lens"])
    out = []
    for i in range(b):
        if case["lens"] == 0 or i == 0:
            n, total = new, top
        else:
            n = _log(r, 1, new)
            total = min(top, n + (_log(r, 1, top - n + 1) - 1 if r.random() < 0.6 or new == 1 else 0))
        out.append((n, total))
    if case["lens"] and b >= 8:
        out[-1] = (1 if new == 1 else 0, 0)
    return out


def _visible(case, pos):
    """How many keys a query at position pos sees."""
    if pos < 0:
        return 0
    w = case.get("window", 0)
    start = max(0, pos - w + 1) if w else 0
    return pos + 1 - start + min(case.get("sinks", 0), start)


def work(case):
    e = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "norm":
        n = case["rows"] * case["d"]
        per = e + (1 if case["fp8"] else e) + (2 * e if case["residual"] else 0)
        return {"bytes": n * per + case["d"] * e + (4 * case["rows"] if case["fp8"] else 0), "flops": 5 * n}
    ls = lengths(case)
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    if case["op"] == "rope":
        tokens = sum(n for n, total in ls if total)
        # q read and written, k and v read and written, the cosines and sines of the positions met
        return {"bytes": tokens * d * e * (2 * hq + 4 * hkv) + min(tokens, case["max_len"]) * d * 4,
                "flops": 3 * tokens * d * (hq + hkv)}
    tokens = sum(n for n, _ in ls)
    pairs, keys = 0, 0
    for n, total in ls:
        pairs += sum(_visible(case, total - n + i) for i in range(n))
        w = case["window"]
        first = max(0, total - n - w + 1) if w else 0  # the oldest key that the first query's window holds
        keys += max(0, total - first) + min(case["sinks"], first)
    return {"bytes": 2 * tokens * hq * d * e + 2 * keys * hkv * d * e, "flops": 4 * pairs * hq * d}


# ----------------------------------------------------------------- the inputs
def _rope_table(positions, d, device):
    """[positions, d] of 32 bits: the cosines in the first half of a row, the sines in the second (base 10000)."""
    inv = 10000.0 ** (-torch.arange(0, d, 2, dtype=torch.float64, device=device) / d)
    a = torch.arange(positions, dtype=torch.float64, device=device)[:, None] * inv
    return torch.cat([a.cos(), a.sin()], dim=1).float()


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def normal(*shape, scale=1.0):
        return torch.randn(shape, generator=g, device=dev, dtype=dt).mul_(scale)

    s = {"case": case}
    if case["op"] == "norm":
        s["x"] = normal(case["rows"], case["d"])
        s["residual"] = normal(case["rows"], case["d"], scale=3.0) if case["residual"] else None
        s["weight"] = (1 + 0.2 * torch.randn(case["d"], generator=g, device=dev)).to(dt)
        return s
    ls = lengths(case)
    b, hq, hkv, d, page = case["batch"], case["hq"], case["hkv"], case["d"], case["page"]
    width = -(-case["max_len"] // page)
    need = [-(-total // page) for _, total in ls]
    pages = max(1, sum(need))
    # pages in no order; entries past a sequence's end are -1
    perm = torch.randperm(pages, generator=g, device=dev).int()
    need_t = torch.tensor(need, device=dev)
    col = torch.arange(width, device=dev)[None, :]
    at = (torch.cumsum(need_t, 0) - need_t)[:, None] + col
    s["block_table"] = torch.where(col < need_t[:, None], perm[at.clamp(max=pages - 1)], -1).int().contiguous()
    s["k_cache"] = normal(pages, hkv, page, d)
    s["v_cache"] = normal(pages, hkv, page, d)
    s["seq_lens"] = torch.tensor([total for _, total in ls], device=dev, dtype=torch.int32)
    starts = [0]
    for n, _ in ls:
        starts.append(starts[-1] + n)
    tokens = starts[-1]
    s["q_start"] = torch.tensor(starts, device=dev, dtype=torch.int32)
    s["most_new"], s["most_len"] = max(n for n, _ in ls), max(1, max(total for _, total in ls))
    s["q"] = normal(tokens, hq, d, scale=1.5)
    if case["op"] == "rope":
        s["k"], s["v"] = normal(tokens, hkv, d), normal(tokens, hkv, d)
        s["rope"] = _rope_table(case["max_len"], d, dev)
    return s


# ------------------------------------------------------------ the plain forms
def _rms_norm(s):
    x, w = s["x"].float(), s["weight"].float()
    h = x if s["residual"] is None else x + s["residual"].float()
    y = h * torch.rsqrt((h * h).mean(dim=1, keepdim=True) + EPS) * w
    out = {} if s["residual"] is None else {"h": h.to(s["x"].dtype)}
    if s["case"]["fp8"]:
        top = y.abs().amax(dim=1, keepdim=True)
        inv = torch.where(top > 0, F8_MAX / top, 0.0)
        out["y"], out["scale"] = (y * inv).clamp(-F8_MAX, F8_MAX).to(F8), (top / F8_MAX).squeeze(1)
    else:
        out["y"] = y.to(s["x"].dtype)
    return out


def _token_places(s):
    """Each token's sequence and position."""
    t = torch.arange(s["q"].shape[0], device=s["q"].device)
    seq = torch.bucketize(t, s["q_start"][1:].long(), right=True)
    n = (s["q_start"][1:] - s["q_start"][:-1]).long()
    return seq, s["seq_lens"].long()[seq] - n[seq] + t - s["q_start"].long()[seq]


def _rope_append(s):
    page, half = s["case"]["page"], s["case"]["d"] // 2
    seq, pos = _token_places(s)
    there = pos >= 0  # a token of an empty slot has no place in the cache
    cs = s["rope"][pos.clamp(min=0)][:, None, :]
    cos, sin = cs[..., :half], cs[..., half:]

    def turn(x):
        a, b = x.float()[..., :half], x.float()[..., half:]
        return torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1).to(x.dtype)

    q = torch.where(there[:, None, None], turn(s["q"]), 0)
    seq, pos, k, v = seq[there], pos[there], turn(s["k"])[there], s["v"][there]
    where = s["block_table"][seq, pos // page].long()
    s["k_cache"][where, :, pos % page] = k
    s["v_cache"][where, :, pos % page] = v
    return {"q": q, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _gathered(s, cache):
    """[batch, kv heads, tokens, d] of a cache in 32 bits, padded to the longest sequence."""
    pages = -(-s["most_len"] // s["case"]["page"])
    x = cache[s["block_table"][:, :pages].clamp(min=0).long()]
    return x.permute(0, 2, 1, 3, 4).flatten(2, 3).float()


def _attention(s):
    case = s["case"]
    b, hq, hkv, d, m = case["batch"], case["hq"], case["hkv"], case["d"], s["most_new"]
    dev = s["q"].device
    n = (s["q_start"][1:] - s["q_start"][:-1]).long()
    i = torch.arange(m, device=dev)
    pos = (s["seq_lens"].long() - n)[:, None] + i  # [batch, new]
    k, v = _gathered(s, s["k_cache"]), _gathered(s, s["v_cache"])
    j = torch.arange(k.shape[2], device=dev)
    seen = (j <= pos[..., None]) & (i < n[:, None])[..., None]  # [batch, new, tokens]
    if case["window"]:
        seen &= (j > pos[..., None] - case["window"]) | (j < case["sinks"])
    v = torch.where((j < s["seq_lens"].long()[:, None])[:, None, :, None], v, 0.0)
    rows = (s["q_start"][:-1].long()[:, None] + i).clamp(max=s["q"].shape[0] - 1)
    q = s["q"][rows].float().view(b, m, hkv, hq // hkv, d).permute(0, 2, 3, 1, 4).reshape(b, hkv, -1, d)
    p = torch.matmul(q, k.transpose(2, 3)).mul_(d ** -0.5).view(b, hkv, hq // hkv, m, -1)
    p = p.masked_fill_(~seen[:, None, None], float("-inf"))
    top = p.amax(dim=-1, keepdim=True)
    p = p.sub_(torch.where(top == float("-inf"), 0.0, top)).exp_()
    total = p.sum(dim=-1, keepdim=True)
    o = torch.matmul(p.view(b, hkv, -1, p.shape[-1]), v).view(b, hkv, hq // hkv, m, d)
    o = torch.where(total > 0, o / total, 0.0).permute(0, 3, 1, 2, 4).reshape(b, m, hq, d)
    seq, at = _token_places(s)
    return o[seq, at - pos[seq, 0]].to(s["q"].dtype)


# ---------------------------------------------------------------- what is run
def run(state):
    s, case = state, state["case"]
    if not own:
        return {"norm": _rms_norm, "rope": _rope_append, "decode": _attention, "prefill": _attention}[case["op"]](s)
    import cube_awq_b200 as cawq
    if case["op"] == "norm":
        if case["fp8"]:
            y, scale, h = cawq.rms_norm_fp8(s["x"], s["weight"], EPS, residual=s["residual"])
            return {"y": y, "scale": scale} if h is None else {"y": y, "scale": scale, "h": h}
        y, h = cawq.rms_norm(s["x"], s["weight"], EPS, residual=s["residual"])
        return {"y": y} if h is None else {"y": y, "h": h}
    if case["op"] == "rope":
        q = cawq.rope_append(s["q"], s["k"], s["v"], s["rope"], s["k_cache"], s["v_cache"], s["block_table"],
                             s["seq_lens"], q_start=None if case["new"] == 1 else s["q_start"])
        return {"q": q, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}
    if case["op"] == "decode":
        return cawq.attention_decode(s["q"], s["k_cache"], s["v_cache"], s["block_table"], s["seq_lens"],
                                     window=case["window"], sinks=case["sinks"])
    return cawq.attention_prefill(s["q"], s["k_cache"], s["v_cache"], s["block_table"], s["seq_lens"], s["q_start"],
                                  window=case["window"], sinks=case["sinks"])


# ----------------------------------------------------- the definition, exactly
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm":
        h = s["x"].double() + (s["residual"].double() if case["residual"] else 0)
        y = h / (h.square().sum(dim=1, keepdim=True) / case["d"] + EPS).sqrt() * s["weight"].double()
        out = {"h": h} if case["residual"] else {}
        if case["fp8"]:
            scale = y.abs().max(dim=1).values / F8_MAX
            return {**out, "y": y / scale[:, None], "scale": scale}
        return {**out, "y": y}
    ls, d, page = lengths(case), case["d"], case["page"]
    if case["op"] == "rope":
        kc, vc = s["k_cache"].double(), s["v_cache"].double()
        q = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
        sign = torch.cat([-torch.ones(d // 2), torch.ones(d // 2)]).double().cuda()
        at = 0
        for i, (n, total) in enumerate(ls):
            rows = slice(at, at + n)
            at += n
            if total == 0 or n == 0:
                continue
            pos = torch.arange(total - n, total, device="cuda")
            cos = s["rope"].double()[pos, : d // 2].repeat(1, 2)[:, None]
            sin = s["rope"].double()[pos, d // 2:].repeat(1, 2)[:, None] * sign
            turn = lambda x: x.double() * cos + x.double().roll(d // 2, dims=-1) * sin  # noqa: E731
            q[rows] = turn(s["q"][rows])
            to = s["block_table"][i].long()[pos // page]
            kc[to, :, pos % page], vc[to, :, pos % page] = turn(s["k"][rows]), s["v"][rows].double()
        return {"q": q, "k_cache": kc, "v_cache": vc}
    group = case["hq"] // case["hkv"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    at = 0
    for i, (n, total) in enumerate(ls):
        rows = slice(at, at + n)
        at += n
        if total == 0 or n == 0:
            continue
        mine = s["block_table"][i, : -(-total // page)].long()
        pos = torch.arange(total - n, total, device="cuda")[:, None]
        key = torch.arange(total, device="cuda")[None, :]
        hidden = key > pos
        if case["window"]:
            hidden |= (pos - key >= case["window"]) & (key >= case["sinks"])
        for h in range(case["hq"]):
            k = s["k_cache"][mine, h // group].reshape(-1, d)[:total].double()
            v = s["v_cache"][mine, h // group].reshape(-1, d)[:total].double()
            score = (s["q"][rows, h].double() @ k.T) / d ** 0.5
            out[rows, h] = torch.softmax(score.masked_fill(hidden, float("-inf")), dim=1) @ v
    return out
