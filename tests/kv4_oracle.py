"""64-bit plain forms that the tests of the rotary, append / read and 4-bit attention kernels compare with (CPU)."""
import math

import torch


def rotate(x, pos, freqs, factor, layout, adjoint=False):
    """x [T,H,D] at positions [T]; freqs: radians per position of each pair (Python floats)."""
    f = torch.tensor(freqs, dtype=torch.float64)
    R = 2 * len(freqs)
    a = pos.double()[:, None, None] * f * (-1.0 if adjoint else 1.0)
    c, s = a.cos() * factor, a.sin() * factor
    y = x.double().clone()
    i = torch.arange(R // 2)
    first, second = (i, i + R // 2) if layout == "half" else (2 * i, 2 * i + 1)
    u, w = x.double()[..., first], x.double()[..., second]
    y[..., first] = u * c - w * s
    y[..., second] = w * c + u * s
    return y


def rotate_slack(x, layout, R, factor):
    """What 32-bit arithmetic may be off by: sine and cosine by 4e-7 (half a step of the argument times pi, two steps of the
    result), each product and the sum by half a step: below 1e-6 of the pair's absolute sum."""
    y = torch.zeros_like(x, dtype=torch.float64)
    i = torch.arange(R // 2)
    first, second = (i, i + R // 2) if layout == "half" else (2 * i, 2 * i + 1)
    both = (x.double()[..., first].abs() + x.double()[..., second].abs()) * factor * 1e-6
    y[..., first] = both
    y[..., second] = both
    return y


def half_step(ref, dtype):
    """Rounding of ref to dtype: half a step relative, and of the smallest subnormal."""
    tiny = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -150}[dtype]
    return ref.abs() * (torch.finfo(dtype).eps / 2) + tiny


def quantise4(x):
    """Codes (int8) and bf16 scales of rows in groups of 32, in 32-bit arithmetic like the kernel's."""
    g = x.float().unflatten(-1, (-1, 32))
    s = (g.abs().amax(-1) / 7).to(torch.bfloat16)
    d = s.float()[..., None]
    c = torch.where(d > 0, g / torch.where(d > 0, d, torch.ones_like(d)), torch.zeros_like(g))
    return c.round().clamp(-7, 7).flatten(-2).to(torch.int8), s


def values4(codes, scale):
    return codes.double() * scale.double().repeat_interleave(32, -1)


def attend(q, k, v, vstep, scale, n_new):
    """q [n,Hq,D], k/v [len,Hkv,D], vstep [len,Hkv,D] (a value's quantisation step); query i sees len - n + i + 1 tokens.

    Returns the output and the bound of the kernel's error before its last rounding: each weight is rounded to fp16
    (2^-11), scores and exponentials are 32-bit (2^-14 covers them at the sizes tested), and value codes are summed as
    code + 8 in 32 bits before the 8 is taken out (2^-17 of 16 steps a weight)."""
    n, Hq, D = q.shape
    length, Hkv = k.shape[:2]
    out = torch.zeros(n, Hq, D, dtype=torch.float64)
    tol = torch.zeros_like(out)
    for i in range(n):
        see = length - n_new + i + 1
        if see <= 0:
            continue
        qi = q[i].double().view(Hkv, -1, D)
        s = torch.einsum("hgd,thd->hgt", qi, k[:see].double()) * scale
        p = torch.softmax(s, -1)
        out[i] = torch.einsum("hgt,thd->hgd", p, v[:see].double()).reshape(Hq, D)
        tol[i] = (torch.einsum("hgt,thd->hgd", p, v[:see].double().abs()) * (2.0 ** -11 + 2.0 ** -14)
                  + torch.einsum("hgt,thd->hgd", p, vstep[:see].double()) * 2.0 ** -13).reshape(Hq, D)
    return out, tol


def ints(*x):
    return torch.tensor(x, dtype=torch.int32)


def offsets(counts):
    return torch.tensor([sum(counts[:i]) for i in range(len(counts) + 1)], dtype=torch.int32)


def page_table(pages, extra, gen):
    """Pages handed out in random order, ``extra`` of the pool unused; entries behind a sequence's pages hold page 0."""
    perm = torch.randperm(sum(pages) + extra, generator=gen).to(torch.int32)
    table = torch.zeros(len(pages), max(1, max(pages)), dtype=torch.int32)
    at = 0
    for b, n in enumerate(pages):
        table[b, :n] = perm[at:at + n]
        at += n
    return table, sum(pages) + extra


def close(got, want, tol):
    got = got.double().cpu()
    bad = (got - want).abs() > tol
    assert not bad.any() and not torch.isnan(got).any(), (
        f"{int(bad.sum())} of {bad.numel()} outside; worst ratio {float(((got - want).abs() / tol).nan_to_num(math.inf).max())}")
