"""The layer operators by their definitions in 64 bits, and error bounds that
follow from how each is computed (fp32 sums, one rounding at the end, softmax
weights rounded once to the operand type)."""

from __future__ import annotations

import torch

# unit roundoff (half a unit in the last place, relative) and the absolute
# error of results in the type's subnormal range
ROUND = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
FLOOR = {torch.float32: 1e-38, torch.float16: 2.0 ** -25, torch.bfloat16: 1e-38}
F32 = 2.0 ** -24


def norm_ref(x, weight, eps, residual=None):
    h = x.double() + (residual.double() if residual is not None else 0)
    y = h / (h.square().mean(dim=-1, keepdim=True) + eps).sqrt() * weight.double()
    return h, y


def norm_rel(d: int) -> float:
    """Relative error of an fp32 y: a sum of d squares over at least 128
    partial sums and their tree, then a root, a quotient and two products."""
    return (-(-d // 128) + 24) * F32


class Cache:
    """A paged cache filled with NaN but for the tokens of its sequences."""

    def __init__(self, seqs, hkv, d, page, dtype, device, seed=0, layout="head", spare=2,
                 evict_window=None, sinks=0, table_extra=1):
        g = torch.Generator(device=device).manual_seed(seed)
        need = [-(-total // page) for _, total in seqs]
        pages = sum(need) + spare
        if layout == "token":      # tokens outermost in a page
            pool = torch.full((2, pages, page, hkv, d), float("nan"), dtype=dtype, device=device)
            self.k, self.v = pool[0].transpose(1, 2), pool[1].transpose(1, 2)
        elif layout == "pair":     # a page's keys and values side by side
            pool = torch.full((pages, 2, hkv, page, d), float("nan"), dtype=dtype, device=device)
            self.k, self.v = pool[:, 0], pool[:, 1]
        else:
            pool = torch.full((2, pages, hkv, page, d), float("nan"), dtype=dtype, device=device)
            self.k, self.v = pool[0], pool[1]
        self.page, self.seqs, self.pages = page, seqs, pages
        width = max([1] + need) + table_extra
        perm = torch.randperm(pages, generator=g, device=device).int()
        table = torch.full((len(seqs), width), -7, dtype=torch.int32, device=device)
        at = 0
        self.kd, self.vd = [], []
        for i, (n, total) in enumerate(seqs):
            mine = perm[at:at + need[i]]
            at += need[i]
            table[i, :need[i]] = mine
            kk = torch.randn((total, hkv, d), generator=g, device=device).to(dtype)
            vv = torch.randn((total, hkv, d), generator=g, device=device).to(dtype)
            self.kd.append(kk)
            self.vd.append(vv)
            pos = torch.arange(total, device=device)
            if total:
                pg = mine.long()[pos // page]
                self.k[pg, :, pos % page] = kk
                self.v[pg, :, pos % page] = vv
            if evict_window and total:  # pages that no query's window holds are given away
                first = max(0, total - max(n, 1) - evict_window + 1)
                for p in range(-(-sinks // page), first // page):
                    table[i, p] = pages + 5
                    self.k[mine[p].long()] = float("nan")
                    self.v[mine[p].long()] = float("nan")
        self.table = table
        self.lens = torch.tensor([total for _, total in seqs], dtype=torch.int32, device=device)
        starts = [0]
        for n, _ in seqs:
            starts.append(starts[-1] + n)
        self.starts = starts
        self.q_start = torch.tensor(starts, dtype=torch.int32, device=device)


def attention_ref(q, cache: Cache, window=0, sinks=0, scale=None):
    """(out, bound) in fp64: the definition, and how far a result may be off."""
    tokens, hq, d = q.shape
    scale = d ** -0.5 if scale is None else scale
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    tol = torch.zeros_like(out)
    u = ROUND[q.dtype]
    for i, (n, total) in enumerate(cache.seqs):
        if n == 0:
            continue
        rows = slice(cache.starts[i], cache.starts[i] + n)
        hkv = cache.k.shape[1]
        k = cache.kd[i].double().repeat_interleave(hq // hkv, dim=1).permute(1, 0, 2)
        v = cache.vd[i].double().repeat_interleave(hq // hkv, dim=1).permute(1, 0, 2)
        pos = (total - n + torch.arange(n, device=q.device))[:, None]
        j = torch.arange(total, device=q.device)[None]
        seen = j <= pos
        if window:
            seen &= (j > pos - window) | (j < sinks)
        qq = q[rows].double().permute(1, 0, 2)
        s = (qq @ k.transpose(1, 2)) * scale
        reach = (qq.abs() @ k.abs().transpose(1, 2)) * abs(scale)
        none = ~seen.any(dim=1)
        s = s.masked_fill(~seen, float("-inf"))
        p = torch.softmax(s, dim=-1) if total else s
        p = torch.where(none[:, None], 0.0, p)
        o = p @ v
        spread = p @ v.abs()
        top = reach.masked_fill(~seen, 0).amax(dim=-1, keepdim=True) if total else 0.0
        small = seen.double() @ v.abs()  # weights below the type's normal range
        count = seen.sum(dim=1).double()[:, None]
        rel = u + 4 * d * F32 * top + (2 * count + 32) * F32
        t = u * o.abs() + rel * spread + 2.0 ** -25 * small * (q.dtype == torch.float16)
        out[rows] = o.permute(1, 0, 2)
        tol[rows] = (t * (1 + u) + FLOOR[q.dtype]).permute(1, 0, 2)
    return out, tol


def assert_within(got, ref, tol, what=""):
    err = (got.double() - ref).abs()
    bad = ~(err <= tol)
    if bool(bad.any()):
        at = int((err / tol.clamp(min=1e-300)).nan_to_num(nan=float("inf")).argmax())
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} off; worst at {at}: got "
                             f"{got.flatten()[at].item()}, want {ref.flatten()[at].item()} +- "
                             f"{tol.flatten()[at].item()}")
