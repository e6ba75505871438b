"""4-bit attention where value scales, values or scores lie far apart: groups of channels of very different size in one row, a
large token that hardly counts, values near the ends of bf16's range, scores far from zero."""
import pytest
import torch

from kv4_oracle import attend, close, half_step, ints, page_table, quantise4, values4
from llm_inference_optimization_b200 import paged

pytestmark = pytest.mark.gpu


class Cache:
    """One kv-head a sequence of the given lengths; ``k`` and ``v`` [tokens, D] of the sequences one behind the other."""

    def __init__(self, k, v, lens, dev):
        D, g = k.shape[1], torch.Generator().manual_seed(1)
        self.lens, self.table = lens, None
        self.table, pages = page_table([(n + 15) // 16 for n in lens], 1, g)
        rows = [torch.zeros(pages, 1, 16, D), torch.zeros(pages, 1, 16, D)]
        at = 0
        for b, n in enumerate(lens):
            t = torch.arange(n)
            for dst, src in zip(rows, (k, v)):
                dst[self.table[b, t // 16].long(), 0, t % 16] = src[at:at + n]
            at += n
        (self.kc, self.ks), (self.vc, self.vs) = (quantise4(x) for x in rows)
        self.kv = paged.PagedKV4(paged.pack_kv4(self.kc, self.ks, self.vc, self.vs).to(dev), self.table.to(dev), ints(*lens).to(dev), len(lens))

    def rows(self, b):
        t = torch.arange(self.lens[b])
        row = lambda x: x.transpose(1, 2)[self.table[b, t // 16].long(), t % 16]  # noqa: E731
        return values4(row(self.kc), row(self.ks)), values4(row(self.vc), row(self.vs)), row(self.vs).double().repeat_interleave(32, -1)

    def check(self, q, scale, dev, dtype):
        """Against the 64-bit formula.  A weight times its value scale has 11 bits (in attend's bound) down to 2^-22 of the largest
        weight times the largest scale of the value's own 32 channels, and is off by at most 2^-33 of that below (half of fp16's
        smallest step, 2^-25, where that product is at least 2^8); codes are at most 7, with the 8 that the kernel takes out
        of them 15."""
        got = self.kv.decode(q.to(dev), scale, out=torch.empty(q.shape, dtype=dtype, device=dev))
        want, tol = [], []
        for b, n in enumerate(self.lens):
            k, v, step = self.rows(b)
            o, t = attend(q[b:b + 1], k, v, step, scale, 1)
            p = torch.softmax(q[b].double() @ k[:, 0].T * scale, -1)                          # [Hq, n]
            tiny = p.amax(-1)[:, None] * step[:, 0].amax(0) * (15 * 2.0 ** -33)                # [Hq, D], a token
            tol.append(t + n * tiny)
            want.append(o)
        want, tol = torch.cat(want), torch.cat(tol)
        close(got, want, tol + half_step(want, dtype))
        return want


def normal(shape, seed):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed))


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Hq", [4, 12])              # 8 and 16 columns a pass
@pytest.mark.parametrize("bits", [20, 34, 60, 100])
def test_groups_of_very_different_size(cuda_device, D, Hq, bits):
    """The channels of one group of 32 are 2^bits times those of another, in every row: each group keeps its own eleven bits."""
    lens = [500, 33]
    v = normal((533, D), 2)
    v[:, 32:64] *= 2.0 ** (bits // 2)
    v[:, :32] *= 2.0 ** -(bits - bits // 2)
    Cache(normal((533, D), 1), v, lens, cuda_device).check(normal((2, Hq, D), 3).half(), D ** -0.5, cuda_device, torch.bfloat16)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("at", [0, 17, 250])
def test_a_large_token_that_hardly_counts(cuda_device, D, at):
    """One value row 2^20 times the others whose weight is below 2^-40: what the others make is kept to the bound stated."""
    k, v = normal((300, D), 4) * 0.1, normal((300, D), 5)
    q = normal((1, 4, D), 6)
    q[..., 0] = 8.0
    k[at, 0] = -40.0                                  # score -320 * scale, the others' within a few units
    v[at] *= 2.0 ** 20
    Cache(k, v, [300], cuda_device).check(q.half(), 0.1, cuda_device, torch.bfloat16)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("power", [-100, -60, 90, 105, 118, 124])
def test_values_near_the_ends_of_the_range(cuda_device, D, power):
    """Neither weights nor sums leave their range where values come near the ends of bf16's."""
    v = normal((2100, D), 7).clamp(-4, 4) * 2.0 ** power
    want = Cache(normal((2100, D), 8), v, [2000, 100], cuda_device).check(normal((2, 8, D), 9).half(), D ** -0.5, cuda_device, torch.bfloat16)
    assert want.abs().max() > 0


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("size", [3e3, 1e5, 1e9, 1e15, 3e15, 1e16])
def test_equal_scores_of_any_size(cuda_device, D, size, sign):
    """Scores from 6e8 to 1e34 of either sign are scores: the softmax over equal ones is their mean."""
    k = torch.full((20, D), sign * size)
    v = normal((20, D), 10)
    q = torch.full((1, 4, D), size).bfloat16()
    c = Cache(k, v, [20], cuda_device)
    want = c.rows(0)[1].mean(0).expand(4, D)          # all scores are equal: D * q * k
    got = c.kv.decode(q.to(cuda_device), 1.0)
    close(got[0], want, c.rows(0)[1].abs().mean(0) * (2.0 ** -11 + 2.0 ** -14) + c.rows(0)[2].mean(0) * 2.0 ** -13 + half_step(want, torch.bfloat16))


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("size", [1e5, 1e9, 1e15])
def test_the_largest_of_large_scores_takes_all(cuda_device, D, size):
    """Scores of 1e11 and more that are apart by a seventh of themselves: the value of the largest comes out, wherever it lies."""
    lens = [300, 300, 17]
    k = torch.full((617, D), size * 6 / 7)
    best = [0, 300 + 299, 600 + 16]
    k[best] = size
    c = Cache(k, normal((617, D), 11), lens, cuda_device)
    q = torch.full((3, 4, D), size).half() if size < 6e4 else torch.full((3, 4, D), size).bfloat16()
    got = c.kv.decode(q.to(cuda_device), 1.0)
    for b in range(3):
        want = c.rows(b)[1][best[b] - sum(lens[:b])].expand(4, D)
        close(got[b], want, want.abs() * (2.0 ** -11 + 2.0 ** -14) + c.rows(b)[2][0] * 2.0 ** -13 + half_step(want, torch.bfloat16))


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("power", [-110, 100, 116, 118, 121, 124])
def test_queries_near_the_ends_of_the_range(cuda_device, D, power):
    """bf16 queries of 2^-110 to 2^125 with a softmax scale that keeps the scores ordinary."""
    q = (normal((2, 8, D), 12).clamp(-3, 3) * 2.0 ** power).bfloat16()
    Cache(normal((133, D), 13), normal((133, D), 14), [100, 33], cuda_device).check(q, D ** -0.5 * 2.0 ** -power, cuda_device, torch.bfloat16)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("bits", [10, 20, 26])
def test_a_large_token_that_only_the_last_query_sees(cuda_device, D, bits):
    """Value scales are bounded over all tokens of the sequence: earlier queries keep to the bound that is stated with them."""
    n, m = 100, 4
    v = normal((n, D), 15)
    v[n - 1] *= 2.0 ** bits
    c = Cache(normal((n, D), 16), v, [n], cuda_device)
    q = normal((m, 4, D), 17).half()
    got = c.kv.decode(q.to(cuda_device), D ** -0.5, cu_q=ints(0, m).to(cuda_device), out=torch.empty(m, 4, D, dtype=torch.bfloat16, device=cuda_device))
    k, values, step = c.rows(0)
    want, tol = attend(q, k, values, step, D ** -0.5, m)
    for i in range(m):
        see = n - m + i + 1
        p = torch.softmax(q[i].double() @ k[:see, 0].T * D ** -0.5, -1)
        tol[i] += see * p.amax(-1)[:, None] * step[:, 0].amax(0) * (15 * 2.0 ** -33)
    close(got, want, tol + half_step(want, torch.bfloat16))
