"""Attention over a cache held in 4 bits, against the 64-bit formula on the dequantised cache."""
import pytest
import torch

from kv4_oracle import attend, close, half_step, ints, offsets, page_table, quantise4, values4
from llm_inference_optimization_b200 import _C, _workspace, paged, rotary

pytestmark = pytest.mark.gpu


class Case:
    """A cache of the given lengths with known codes and scales, and queries for it."""

    def __init__(self, lens, queries, Hq, Hkv, D, dtype, dev, seed=0, unit=1.0, capacity=None, spread=0.0, table=True):
        g = torch.Generator().manual_seed(seed)
        self.lens, self.queries, self.dev, self.B = lens, queries, dev, len(lens)
        pages = [max((n + 15) // 16, 0) for n in lens]
        if table:
            self.table, self.pages = page_table(pages, 3, g)
        else:
            per = max(max(pages), 1)
            self.pages = per * self.B
            self.table = torch.arange(self.pages, dtype=torch.int32).view(self.B, per)
        if capacity:
            self.table = torch.cat([self.table, torch.zeros(self.B, capacity - self.table.shape[1], dtype=torch.int32)], 1)
        shape = (self.pages, Hkv, 16, D)
        mul = torch.exp2(spread * torch.randn(*shape[:3], 1, generator=g))
        self.k, self.ks = quantise4(torch.randn(shape, generator=g) * unit)
        self.v, self.vs = quantise4(torch.randn(shape, generator=g) * mul)
        self.q = (torch.randn(sum(queries), Hq, D, generator=g)).to(dtype)
        self.buf = paged.pack_kv4(self.k, self.ks, self.v, self.vs).to(dev)
        self.kv = paged.PagedKV4(self.buf, self.table.to(dev) if table else None, ints(*lens).to(dev), self.B)
        self.cu = None if set(queries) == {1} else offsets(queries).to(dev)
        self.scale = D ** -0.5

    def rows(self, b):
        n = self.lens[b]
        t = torch.arange(n)
        at = lambda x: x.transpose(1, 2)[self.table[b, t // 16].long(), t % 16]  # noqa: E731
        k, v = values4(at(self.k), at(self.ks)), values4(at(self.v), at(self.vs))
        return k, v, at(self.vs).double().repeat_interleave(32, -1)

    def want(self):
        out, tol, at = [], [], 0
        for b, m in enumerate(self.queries):
            o, t = attend(self.q[at:at + m], *self.rows(b), self.scale, m)
            out.append(o)
            tol.append(t)
            at += m
        return torch.cat(out), torch.cat(tol)

    def check(self, got=None, dtype=None):
        got = self.run() if got is None else got
        want, tol = self.want()
        close(got, want, tol + half_step(want, got.dtype))
        return got

    def run(self, **kw):
        return self.kv.decode(self.q.to(self.dev), self.scale, cu_q=self.cu, **kw)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("n", [0, 1, 2, 15, 16, 17, 63, 128, 129, 1000, 4099])
def test_one_sequence(cuda_device, D, dtype, n):
    got = Case([n], [1], 8, 2, D, dtype, cuda_device, seed=n).check()
    if n == 0:
        assert (got == 0).all()


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Hkv,G", [(1, 1), (2, 3), (1, 8), (3, 5), (1, 9), (2, 16), (1, 32), (8, 4)])
def test_head_groups(cuda_device, D, Hkv, G):
    Case([300, 0, 77, 1], [1, 1, 1, 1], Hkv * G, Hkv, D, torch.float16, cuda_device, seed=G).check()


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("queries", [[4, 4, 4], [1, 0, 7], [16, 2, 3], [0, 0, 1], [33, 5, 64]])
def test_several_queries_are_causal(cuda_device, D, queries):
    Case([500, 16, 65], queries, 8, 2, D, torch.bfloat16, cuda_device, seed=sum(queries)).check()


def test_more_queries_than_tokens_see_nothing_first(cuda_device):
    c = Case([3, 0, 20], [5, 2, 20], 4, 2, 64, torch.float16, cuda_device)
    got = c.check()
    assert (got[:2] == 0).all() and (got[5:7] == 0).all() and (got[2] != 0).any()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_long_contexts_split_over_many_blocks(cuda_device, dtype):
    Case([40001, 70, 9000], [1, 1, 1], 4, 1, 128, dtype, cuda_device, seed=1).check()
    Case([33333], [3], 4, 1, 64, dtype, cuda_device, seed=2).check()


def test_many_sequences(cuda_device):
    lens = [(i * 53) % 170 for i in range(150)]
    Case(lens, [1] * 150, 4, 2, 64, torch.float16, cuda_device, seed=3).check()
    Case(lens, [(i * 5) % 4 for i in range(150)], 4, 2, 64, torch.float16, cuda_device, seed=4).check()


def test_without_page_table_and_lengths(cuda_device):
    c = Case([64, 64], [1, 1], 4, 2, 64, torch.float16, cuda_device, table=False)
    c.check()
    full = paged.PagedKV4(c.buf, None, None, 2).decode(c.q.to(cuda_device), c.scale)
    assert torch.equal(full, c.run())
    c.lens = [50, 50]                                # max_seq_len bounds sequences without lengths
    c.check(paged.PagedKV4(c.buf, None, None, 2).decode(c.q.to(cuda_device), c.scale, max_seq_len=50))
    c.lens = [40, 40]                                # and clamps lengths beyond it
    c.check(paged.PagedKV4(c.buf, None, ints(64, 64).to(cuda_device), 2).decode(c.q.to(cuda_device), c.scale, max_seq_len=40))


@pytest.mark.parametrize("spread", [4.0, 12.0])
def test_value_scales_of_very_different_size(cuda_device, spread):
    """Rows a few thousand times larger or smaller than others: weights keep their eleven bits relative to what counts."""
    Case([700, 30], [1, 1], 8, 2, 128, torch.bfloat16, cuda_device, seed=5, spread=spread).check()


@pytest.mark.parametrize("size", [2.0 ** -20, 1e-4, 300.0, 30000.0])
def test_queries_and_keys_of_any_size(cuda_device, size):
    c = Case([200, 33], [1, 1], 8, 2, 64, torch.float16 if size < 1 else torch.bfloat16, cuda_device, seed=6, unit=1.0)
    c.q = (c.q.float() * size).to(c.q.dtype)
    c.scale = 64 ** -0.5 / size                      # the scores stay ordinary
    c.check()


def test_sharp_softmax_and_rows_of_zeros(cuda_device):
    c = Case([300], [1], 4, 1, 128, torch.float16, cuda_device, seed=7, unit=1.0)
    c.scale = 1.0                                    # scores of tens: one token takes nearly all
    c.check()
    c.vs[:] = 0
    c.v[:] = 0
    c.buf.copy_(paged.pack_kv4(c.k, c.ks, c.v, c.vs))
    assert (c.run() == 0).all()


def test_garbage_behind_the_end_is_not_seen(cuda_device):
    """Records behind a sequence's last token may hold anything: scales of NaN and infinity, codes of all ones."""
    for D in (64, 128):
        c = Case([37, 16, 1], [1, 3, 1], 8, 2, D, torch.float16, cuda_device, seed=8)
        want = c.run()
        for b, n in enumerate(c.lens):
            for t in range(n, (n + 15) // 16 * 16):
                page = int(c.table[b, t // 16])
                c.k[page, :, t % 16], c.v[page, :, t % 16] = -8 + 15, -8 + 15
                c.ks[page, :, t % 16] = float("nan")
                c.vs[page, :, t % 16] = float("nan") if t % 2 else float("inf")
        c.buf.copy_(paged.pack_kv4(c.k, c.ks, c.v, c.vs))
        assert torch.equal(c.run(), want)


def test_not_a_number_reaches_those_who_see_it_only(cuda_device):
    c = Case([40, 40], [4, 1], 4, 1, 128, torch.float16, cuda_device, seed=9)
    want = c.run()
    page, slot = int(c.table[0, 38 // 16]), 38 % 16   # token 38 is seen by the queries at 38 and 39
    c.vs[page, 0, slot, 1] = float("nan")
    c.buf.copy_(paged.pack_kv4(c.k, c.ks, c.v, c.vs))
    got = c.run()
    assert torch.equal(got[[0, 1, 4]], want[[0, 1, 4]])
    nan = torch.isnan(got[2:4]).cpu()
    assert nan[..., 32:64].all() and not nan[..., :32].any() and not nan[..., 64:].any()
    c.vs[page, 0, slot, 1] = 1.0
    c.ks[page, 0, slot, 0] = float("nan")
    c.buf.copy_(paged.pack_kv4(c.k, c.ks, c.v, c.vs))
    got = c.run()
    assert torch.isnan(got[2:4]).all() and torch.equal(got[[0, 1, 4]], want[[0, 1, 4]])


def test_rows_behind_the_last_sequence_and_given_outputs(cuda_device):
    c = Case([100, 30], [2, 3], 4, 2, 64, torch.bfloat16, cuda_device, seed=10)
    want, tol = c.want()
    q = torch.cat([c.q, torch.zeros(4, 4, 64, dtype=c.q.dtype)]).to(cuda_device)
    for dtype in (torch.float16, torch.bfloat16):
        out = torch.full(q.shape, 55.0, dtype=dtype, device=cuda_device)
        assert c.kv.decode(q, c.scale, cu_q=c.cu, out=out) is out
        close(out[:5], want, tol + half_step(want, dtype))
        assert (out[5:] == 55.0).all()


@pytest.mark.parametrize("bad", [-1, 1 << 20, 2 ** 31 - 1])
def test_bad_page_is_reported_and_others_untouched(cuda_device, bad):
    c = Case([100, 30], [1, 1], 4, 2, 64, torch.float16, cuda_device, seed=11)
    want = c.run()
    ws = _workspace.get("gqa_kv4", 0, cuda_device)
    assert _workspace.status(ws) == 0
    c.kv.page_table[1, 1] = bad
    try:
        got = c.run()
        assert _workspace.status(ws) == 2 and torch.equal(got[0], want[0]) and torch.isfinite(got).all()
    finally:
        ws[:4].zero_()
    word = torch.zeros(1, dtype=torch.int32, device=cuda_device)   # a word of the caller's, which a captured call can report to
    q = c.q.to(cuda_device)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.kv.decode(q, c.scale, status=word)
    assert int(word) == 0
    graph.replay()
    assert int(word) == 2 and _workspace.status(ws) == 0


def test_same_bits_every_time_and_on_other_streams(cuda_device):
    c = Case([20000, 3, 5000, 777], [1] * 4, 8, 2, 128, torch.bfloat16, cuda_device, seed=12)
    want = c.check()
    for _ in range(10):
        assert torch.equal(c.run(), want)
    streams = [torch.cuda.Stream() for _ in range(3)]
    outs = []
    torch.cuda.synchronize()
    for _ in range(5):
        for s in streams:
            with torch.cuda.stream(s):
                outs.append(c.run())
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


def test_two_graphs_replayed_at_once(cuda_device):
    cases = [Case([9000, 40], [1, 1], 8, 2, 128, torch.float16, cuda_device, seed=13), Case([6000, 3000], [1, 1], 8, 2, 128, torch.float16, cuda_device, seed=14)]
    want = [c.check() for c in cases]
    graphs, outs, qs = [], [], [c.q.to(cuda_device) for c in cases]
    for c, q in zip(cases, qs):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append([c.kv.decode(q, c.scale) for _ in range(3)])
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in graphs]
    torch.cuda.synchronize()
    for _ in range(10):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        eager = cases[0].run()
    torch.cuda.synchronize()
    assert torch.equal(eager, want[0])
    for o, w in zip(outs, want):
        assert all(torch.equal(x, w) for x in o)


def test_pool_beyond_four_gigabytes(cuda_device):
    """Page offsets pass 32 bits: the pages in use lie at the end of a 5 GB pool."""
    c = Case([100, 30], [1, 1], 4, 2, 128, torch.float16, cuda_device, seed=15)
    want = c.run()
    total = 5 * 2 ** 30 // (2 * 2304)
    big = torch.empty(total, 2, 18, 128, dtype=torch.uint8, device=cuda_device)
    first = total - c.pages
    big[first:] = c.buf
    kv = paged.PagedKV4(big, c.kv.page_table + first, c.kv.seq_lens, 2)
    assert torch.equal(kv.decode(c.q.to(cuda_device), c.scale), want)
    qkv = torch.randn(2, 8 * 128, generator=torch.Generator().manual_seed(0)).half().to(cuda_device)
    paged.append_tokens(qkv, kv, 4)                  # positions 100 and 30, inside pages in use
    small = paged.PagedKV4(c.buf, c.kv.page_table, c.kv.seq_lens, 2)
    paged.append_tokens(qkv, small, 4)
    assert torch.equal(big[first:], c.buf)
    cu = offsets([101, 31]).to(cuda_device)
    for a, b in zip(paged.read_tokens(kv, cu, 132), paged.read_tokens(small, cu, 132)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("D,layout,dtype", [(128, "half", torch.bfloat16), (64, "interleaved", torch.float16)])
def test_prompt_drafts_and_steps_together(cuda_device, D, layout, dtype):
    """A prompt in two chunks, drafted tokens, single steps: every attention result against the formula on what the cache
    holds, whose rows are read back and compared with the projections."""
    Hq, Hkv, B = 8, 2, 3
    g = torch.Generator().manual_seed(D)
    table, total = page_table([20, 20, 20], 4, g)
    kv = paged.PagedKV4(torch.full((total, Hkv, 18, D), 255, dtype=torch.uint8, device=cuda_device), table.to(cuda_device),
                        torch.zeros(B, dtype=torch.int32, device=cuda_device), B)
    rope = rotary.RotaryEmbedding(D, 10000.0, rotary_dim=D // 2, layout=layout, device=cuda_device)
    lens = [0] * B
    for new in ([40, 0, 100], [3, 17, 130], [4, 4, 2], [1, 1, 1], [1, 1, 1]):
        T = sum(new)
        qkv = torch.randn(T, (Hq + 2 * Hkv) * D, generator=g).to(dtype).to(cuda_device)
        cu = offsets(new).to(cuda_device)
        q = paged.append_tokens(qkv, kv, Hq, rope, cu_new=cu, q_out=torch.empty(T, Hq, D, dtype=dtype, device=cuda_device))
        lens = [a + n for a, n in zip(lens, new)]
        kv.seq_lens += ints(*new).to(cuda_device)
        out = kv.decode(q, D ** -0.5, cu_q=None if set(new) == {1} else cu)
        k, ks, v, vs = (t.cpu() for t in paged.unpack_kv4(kv.buf))
        at = 0
        for b, n in enumerate(new):
            t = torch.arange(lens[b])
            row = lambda x: x.transpose(1, 2)[table[b, t // 16].long(), t % 16]  # noqa: E731,B023
            want, tol = attend(q[at:at + n].cpu(), values4(row(k), row(ks)), values4(row(v), row(vs)),
                               row(vs).double().repeat_interleave(32, -1), D ** -0.5, n)
            close(out[at:at + n], want, tol + half_step(want, dtype))
            at += n
        K, V = paged.read_tokens(kv, cu, T, starts=kv.seq_lens - ints(*new).to(cuda_device), dtype=dtype)
        turned = rope.apply(torch.cat([torch.arange(a - n, a, dtype=torch.int32) for a, n in zip(lens, new)]).to(cuda_device),
                            qkv.view(T, -1, D)[:, Hq:Hq + Hkv].float())
        for got, x in ((K, turned), (V, qkv.view(T, -1, D)[:, Hq + Hkv:].float())):
            step = x.unflatten(-1, (-1, 32)).abs().amax(-1).repeat_interleave(32, -1) / 7
            # half a step of codes made with a scale off by 2^-8, and the rounding of the value read
            assert ((got.float() - x).abs() <= step * (0.5 + 2.0 ** -8) + x.abs() * torch.finfo(dtype).eps + 1e-6).all()


def test_refusals(cuda_device):
    c = Case([32, 20], [1, 1], 4, 2, 64, torch.float16, cuda_device)
    q, cu = c.q.to(cuda_device), offsets([1, 1]).to(cuda_device)
    call = lambda q=q, pool=c.buf, t=c.kv.page_table, n=c.kv.seq_lens, s=0.125, **kw: _C.fused_gqa_kv4(q, pool, t, n, s, **kw)  # noqa: E731
    call()
    for bad in [lambda: call(q=q.float()), lambda: call(q=q[:1]), lambda: call(q=q[:, :3].contiguous()), lambda: call(q=q.transpose(0, 1)),
                lambda: call(q=q[..., :32].contiguous()), lambda: call(pool=c.buf.view(torch.int8)), lambda: call(pool=c.buf[:, :, :17]),
                lambda: call(t=c.kv.page_table.long()), lambda: call(n=c.kv.seq_lens[:1]), lambda: call(n=c.kv.seq_lens.cpu()),
                lambda: call(s=0.0), lambda: call(s=float("nan")), lambda: call(max_seq_len=0), lambda: call(max_seq_len=33),
                lambda: call(cu_q=cu[:2]), lambda: call(cu_q=cu.long()), lambda: call(out=torch.empty_like(q).float()),
                lambda: call(out=torch.empty_like(q)[:1]), lambda: call(q=q.cpu()), lambda: call(status=torch.zeros(2, device=cuda_device)), lambda: call(t=None, pool=c.buf[:3])]:
        with pytest.raises(RuntimeError):
            bad()
