"""The operators around attention written out in 64 bits, sequence by sequence, with bounds on what the kernels' roundings can
make of them.  Used by the tests of rotary positions and of the paged cache."""

import math

import torch


def turned(x, positions, rotary, inverse=False):
    """x [..., N, D] at positions [N], each pair as a complex number, in 64 bits."""
    x = x.detach().double().clone()
    if rotary is None:
        return x
    rd = rotary.rotary_dim
    angle = positions.double()[:, None] * torch.tensor(rotary.frequencies, dtype=torch.float64, device=x.device)
    e = rotary.attention_factor * torch.exp(1j * (-angle if inverse else angle))
    a, b = (slice(0, rd, 2), slice(1, rd, 2)) if rotary.interleaved else (slice(0, rd // 2), slice(rd // 2, rd))
    z = torch.complex(x[..., a], x[..., b]) * e
    x[..., a], x[..., b] = z.real, z.imag
    return x


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


class Sequences:
    """Pages of a batch in random order, with entries behind a sequence that are no pages."""

    def __init__(self, lengths, page_size, extra_pages=3, room=None, seed=0, behind=-7, device="cuda"):
        gen = torch.Generator().manual_seed(seed)
        used = [-(-n // page_size) for n in lengths]
        self.pages, self.page_size = sum(used) + extra_pages, page_size
        order = torch.randperm(self.pages, generator=gen)
        self.table = torch.full((len(lengths), room or max(1, *used)), behind, dtype=torch.int32)
        at = 0
        for b, n in enumerate(used):
            self.table[b, :n] = order[at : at + n]
            at += n
        self.table = self.table.to(device)
        self.lengths = torch.tensor(lengths, dtype=torch.int32, device=device)

    def rows(self, t, b, n):
        """Rows 0 ... n - 1 of sequence b of a cache tensor [P, H, page, X], as [H, n, X]."""
        at = torch.arange(n, device=t.device)
        return t[self.table[b].long()[at // self.page_size], :, at % self.page_size].transpose(0, 1)


def values(cache, which, seqs, b, n):
    """Cached rows in 64 bits."""
    x = seqs.rows(getattr(cache, which), b, n)
    if cache.bits == 16:
        return x.double(), None
    sc = seqs.rows(getattr(cache, which + "_scales"), b, n).double()
    y = torch.stack((x % 16, x // 16), -1).flatten(-2).double()
    return y * sc[..., :1] + sc[..., 1:], sc[..., :1]


def attention(q, cache, seqs, counts=None, *, is_causal=True, scale=None, window_size=0, rotary=None, unpacked=False):
    """(out, bound): attention over the cache in 64 bits, and how far the kernels may be from it.

    Roundings to u = half a step of the type: the result, u |out|; every probability (relative to the row's sum), u sum p |v|,
    in 4 bits u(bf16) sum p 8 step on the part of the values that goes through the product; a query turned on the way,
    which moves a score by at most d = u scale |q| . |k| and the result by (e^(2 d) - 1) (sum p |v| + |out|).
    unpacked: 4-bit rows that are rounded to 16 bits first.  An element is off by u of it at most, thus a score by u scale |q| . |k|,
    as a turned query's, and the result by u sum p |v| more.
    Sums in fp32: scores of D products (in 4 bits with an offset of 128 or 1024 on every code) and the result's sums, 2^-23
    of the sum of magnitudes for each of the D / 16 + 1 steps; the exponential 2^-21.
    """
    B, Hq, N, D = q.shape
    G = Hq // cache.kv_heads
    tau = D ** -0.5 if scale is None else scale
    u = half_step(q.dtype)
    out = torch.zeros(B, Hq, N, D, dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(out)
    for b in range(B):
        n = int(seqs.lengths[b])
        c = N if counts is None else int(counts[b])
        if not n or not c:
            continue
        k, _ = values(cache, "k", seqs, b, n)
        v, step = values(cache, "v", seqs, b, n)
        _, kstep = values(cache, "k", seqs, b, n)
        position = torch.arange(n - c, n, device=q.device)
        distance = position[:, None] - torch.arange(n, device=q.device)
        keep = torch.ones_like(distance, dtype=torch.bool)
        if is_causal:
            keep = distance >= 0
        if window_size:
            keep &= distance < window_size
        k, v = torch.nan_to_num(k), torch.nan_to_num(v)
        x = turned(q[b, :, :c], position, rotary)
        for h in range(Hq):
            kh, vh = k[h // G], v[h // G]
            s = (x[h] @ kh.T * tau).masked_fill(~keep, -math.inf)
            p = torch.softmax(s, -1)
            out[b, h, :c] = p @ vh
            mag = p @ vh.abs()
            size = (x[h].abs() @ kh.abs().T * tau).masked_fill(~keep, 0).amax(-1, keepdim=True)
            d = size * ((u if rotary is not None else 0) + (u if unpacked else 0) + 2.0 ** -23 * (D / 16 + 1))
            if cache.bits == 4:
                off = 128 if q.dtype == torch.bfloat16 else 1024
                d = d + tau * x[h].abs().sum(-1, keepdim=True) * kstep[h // G].max() * (off + 16) * 2.0 ** -23 * (D / 16 + 1)
                mag = mag + 8 * p @ step[h // G]
                up = half_step(torch.bfloat16)
            else:
                up = u
            d = d + 2.0 ** -21
            bound[b, h, :c] = u * out[b, h, :c].abs() + (up + (u if unpacked else 0) + 2.0 ** -20) * mag + torch.expm1(2 * d) * (mag + out[b, h, :c].abs())
    return out, bound


def close(got, want, bound, tiny):
    """Within the bound everywhere (`tiny`: the smallest step of the type, where results underflow)."""
    off = (got.double() - want).abs()
    bad = ~(off <= bound + tiny)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, by up to {float((off / (bound + tiny)).nan_to_num(9e9).max()):.3g} bounds at {bad.nonzero()[0].tolist()}"
