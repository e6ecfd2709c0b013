"""A cache of 8 bits written out plainly, in 64 bits: what the kernels of ``csrc/scaled_*`` are compared with."""

import torch

BLOCK = 16


def exponent_for(largest: torch.Tensor) -> torch.Tensor:
    """The smallest e in -110 .. 118 with 448 * 2^e >= largest."""
    e = torch.full(largest.shape, -110, dtype=torch.int64)
    for k in range(-110, 118):
        e = torch.where(largest > 448.0 * 2.0**k, k + 1, e)
    return e


def to_code(x: torch.Tensor) -> torch.Tensor:
    """The value of the 8-bit code nearest to x (|x| <= 448), ties to even: steps of 2^-3 of the leading power, none below 2^-9."""
    step = 2.0 ** (torch.floor(torch.log2(x.abs().clamp(min=2.0**-6))) - 3)
    return torch.round(x / step) * step


def coded(values: torch.Tensor, e: torch.Tensor) -> torch.Tensor:
    """values * 2^-e as codes (float64); infinities become NaN, larger numbers 448."""
    out = to_code((values.double() * 2.0 ** (-e.double())).clamp(-448.0, 448.0))
    return torch.where(torch.isfinite(values), out, torch.nan)


class PlainPlane:
    """One plane (keys or values): codes as float64 [num_pages, heads, page, size] and exponents [num_pages, heads, page / 16]."""

    def __init__(self, num_pages, heads, page, size):
        self.page = page
        self.codes = torch.zeros((num_pages, heads, page, size), dtype=torch.float64)
        self.e = torch.zeros((num_pages, heads, page // BLOCK), dtype=torch.int64)

    def append(self, rows: torch.Tensor, slots):
        """rows [n, heads, size]; the rule of kernels.scaled_append, a run at a time."""
        slots = [int(s) for s in slots]
        limit = self.codes.shape[0] * self.page
        at = 0
        while at < len(slots):
            end = at + 1
            while end < len(slots) and 0 <= slots[at] < limit and slots[end] == slots[end - 1] + 1 and slots[end] // BLOCK == slots[at] // BLOCK:
                end += 1
            if 0 <= slots[at] < limit:
                page, lead, block = slots[at] // self.page, slots[at] % BLOCK, slots[at] % self.page // BLOCK
                new = rows[at:end].double().transpose(0, 1)                                     # [heads, run, size]
                size = torch.where(torch.isfinite(new), new.abs(), 0.0).amax((1, 2))
                need, old = exponent_for(size), self.e[page, :, block]
                e = torch.maximum(need, old) if lead else need
                lo = block * BLOCK
                if lead:
                    grown = 2.0 ** (old - e).double()[:, None, None]
                    self.codes[page, :, lo : lo + lead] = to_code(self.codes[page, :, lo : lo + lead] * grown)
                self.codes[page, :, lo + lead : lo + lead + end - at, : new.shape[2]] = coded(new, e[:, None, None])
                self.codes[page, :, lo + lead : lo + lead + end - at, new.shape[2] :] = 0.0
                self.e[page, :, block] = e
            at = end

    def held(self) -> torch.Tensor:
        """[num_pages, heads, page, size]: the numbers."""
        return self.codes * 2.0 ** self.e.double().repeat_interleave(BLOCK, dim=-1)[..., None]


def laid(plane: PlainPlane, keys: bool, device):
    """(codes, scales) as kernels.ScaledPages holds them."""
    pages, heads, page, size = plane.codes.shape
    codes = plane.codes.float().to(torch.float8_e4m3fn).view(torch.uint8).view(pages, heads, page // BLOCK, BLOCK, size)
    if keys:
        codes = codes.view(pages, heads, page // BLOCK, BLOCK, size // 16, 16).transpose(3, 4)
    else:
        codes = codes.transpose(3, 4)
    return codes.contiguous().view(torch.float8_e4m3fn).to(device), (2.0 ** plane.e.double()).float().to(device)


def turned(x, positions, frequencies, dims, pairing, sign=1.0):
    """x [rows, heads, size] in float64, the first ``dims`` elements turned in pairs."""
    if not dims:
        return x
    angle = sign * positions.double()[:, None, None] * frequencies.double()[None, None, : dims // 2]
    c, s = torch.cos(angle), torch.sin(angle)
    first = torch.arange(dims // 2) if pairing == "half" else 2 * torch.arange(dims // 2)
    second = first + (dims // 2 if pairing == "half" else 1)
    y = x.clone()
    y[..., first] = x[..., first] * c - x[..., second] * s
    y[..., second] = x[..., second] * c + x[..., first] * s
    return y


def normed(x, gain, eps):
    """RMS norm over the last dimension."""
    y = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
    return y if gain is None else y * gain.double()


def attended(q, k_held, v_held, requests, positions, tables, scale, *, window=0, keep=0, chunk=0, softcap=0.0, sinks=None):
    """q [rows, heads, size], held [num_pages, kv heads, page, size] -> [rows, heads, size], float64; rows that see nothing are zeros."""
    n, heads, size = q.shape
    kv_heads, page = k_held.shape[1], k_held.shape[2]
    out = torch.zeros((n, heads, size), dtype=torch.float64)
    for r in range(n):
        p, b = int(positions[r]), int(requests[r])
        if p < 0 or b < 0:
            continue
        keys = torch.arange(p + 1)
        low = p - p % chunk if chunk else max(0, p - window + 1) if window else 0
        keys = keys[(keys >= low) | (keys < (keep if window else 0))]
        pages = tables[b].long()[keys // page]
        k, v = k_held[pages, :, keys % page], v_held[pages, :, keys % page]                     # [keys, kv heads, size]
        k, v = (t.repeat_interleave(heads // kv_heads, dim=1) for t in (k, v))
        s = torch.einsum("hd,khd->hk", q[r].double(), k) * scale
        if softcap:
            s = softcap * torch.tanh(s / softcap)
        if sinks is not None:
            s = torch.cat([s, sinks.double()[:, None]], dim=1)
        w = torch.softmax(s, dim=1)[:, : len(keys)]
        out[r] = torch.einsum("hk,khd->hd", w, v)
    return out
