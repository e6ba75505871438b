"""Append, read-back and attention where a batch's offsets are unusual: offsets that begin above zero (part of a batch), offsets
that do not ascend; every buffer lies between bytes that must stay as they are."""
import pytest
import torch

from kv4_oracle import ints, offsets, page_table
from llm_inference_optimization_b200 import _lib, _workspace, paged
from llm_inference_optimization_b200 import decode_step as ds
from test_kv_tokens_gpu import FORMATS, empty_cache

pytestmark = pytest.mark.gpu
MARK = 0xA5


def guarded(shape, dtype, dev, raws):
    """A tensor of MARK bytes with 4096 more of them on either side."""
    n = int(torch.tensor(shape).prod()) * torch.empty((), dtype=dtype).element_size()
    raw = torch.full((n + 8192,), MARK, dtype=torch.uint8, device=dev)
    raws.append(raw)
    return raw[4096:4096 + n].view(dtype).view(shape)


def untouched(raws):
    return all(bool((r[:4096] == MARK).all() and (r[-4096:] == MARK).all()) for r in raws)


def read_into(kv, cu, starts, K, V):
    """``paged.read_tokens`` into given buffers, so that rows which are not written can be told."""
    pools, layout, table, Hkv, D, dev = paged._token_cache(kv)
    rc = _lib.load().skv_read_tokens(*pools, table, cu.data_ptr(), starts.data_ptr(), K.data_ptr(), V.data_ptr(), 0, K.shape[0], kv.batch,
                                     Hkv, D, *layout, None, dev.index, _workspace.stream(dev.index))
    _lib.check(rc, "read_tokens")


def cache_bytes(kv):
    return [t.view(torch.uint8) for t in ((kv.buf,) if isinstance(kv, paged.PagedKV4) else (kv.k_pool, kv.v_pool, kv.k_scale, kv.v_scale))]


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("B,first", [(2, 3), (300, 5)])      # counted by all lanes of a row; searched
def test_rows_before_the_first_offset_belong_to_nobody(cuda_device, fmt, B, first):
    """Part of a batch: its offsets begin above zero, and the rows before them change no cached token, no query row, no row read."""
    Hq, Hkv, D = 2, 2, 128
    g = torch.Generator().manual_seed(B)
    old, new = [100 + i % 7 for i in range(B)], [2 + i % 3 for i in range(B)]
    size = 48 if fmt == "pools" else 16
    table, total = page_table([(a + n + size - 1) // size for a, n in zip(old, new)], 0, g)
    part, whole = (empty_cache(fmt, total, Hkv, D, table, ints(*old), B, cuda_device) for _ in range(2))
    T = first + sum(new)
    qkv = torch.randn(T, (Hq + 2 * Hkv) * D, generator=g).half().to(cuda_device)
    cu = (offsets(new) + first).to(cuda_device)
    raws = []
    q = paged.append_tokens(qkv, part, Hq, cu_new=cu, q_out=guarded((T, Hq, D), torch.float16, cuda_device, raws))
    want = paged.append_tokens(qkv[first:], whole, Hq, cu_new=cu - first)
    assert torch.equal(q[first:], want) and (q[:first].view(torch.uint8) == MARK).all()
    assert all(torch.equal(a, b) for a, b in zip(cache_bytes(part), cache_bytes(whole)))
    K, V = (guarded((T, Hkv, D), torch.float16, cuda_device, raws) for _ in range(2))
    read_into(part, cu, part.seq_lens, K, V)
    for got, rows in zip((K, V), paged.read_tokens(whole, cu - first, T - first, starts=whole.seq_lens)):
        assert torch.equal(got[first:], rows) and (got[:first].view(torch.uint8) == MARK).all()
    assert untouched(raws)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("cu", [(5, 2, 9, 1), (-7, 100, -100, 3), (2 ** 31 - 1, -2 ** 31, 0, 9), (9, 9, 9, 0)])
def test_offsets_that_do_not_ascend_write_nothing_else(cuda_device, D, cu):
    """Whatever sequence a row is given, it lands in a page of the table: pages that no sequence owns and the bytes around every
    buffer stay."""
    raws = []
    table, total = page_table([3, 3, 3], 4, torch.Generator().manual_seed(4))
    buf = guarded((total, 2, 18, D), torch.uint8, cuda_device, raws)
    kv = paged.PagedKV4(buf, table.to(cuda_device), ints(0, 0, 0).to(cuda_device), 3)
    qkv = torch.randn(9, 6 * D, generator=torch.Generator().manual_seed(3)).half().to(cuda_device)
    at = ints(*cu).to(cuda_device)
    half = lambda *s: guarded(s, torch.float16, cuda_device, raws)  # noqa: E731
    paged.append_tokens(qkv, kv, 2, cu_new=at, q_out=half(9, 2, D))
    read_into(kv, at, kv.seq_lens, half(9, 2, D), half(9, 2, D))
    kv.decode(torch.randn(9, 2, D, device=cuda_device).half(), 0.125, cu_q=at, out=half(9, 2, D))
    torch.cuda.synchronize()
    assert untouched(raws)
    unowned = sorted(set(range(total)) - set(table.flatten().tolist()))
    assert len(unowned) == 4 and (buf[unowned] == MARK).all()


@pytest.mark.parametrize("D", [64, 128])
def test_attention_of_part_of_a_batch(cuda_device, D):
    raws, g = [], torch.Generator().manual_seed(D)
    table, total = page_table([20, 3], 0, g)
    kv = empty_cache("kv4", total, 2, D, table, ints(0, 0), 2, cuda_device)
    new = [300, 40]
    paged.append_tokens(torch.randn(340, 4 * D, generator=g).half().to(cuda_device), kv, 0, cu_new=offsets(new).to(cuda_device))
    kv.seq_lens += ints(*new).to(cuda_device)
    q = torch.randn(12, 8, D, generator=g).half().to(cuda_device)
    cu = ints(3, 7, 9).to(cuda_device)
    out = kv.decode(q, D ** -0.5, cu_q=cu, out=guarded((12, 8, D), torch.float16, cuda_device, raws))
    assert torch.equal(out[3:9], kv.decode(torch.roll(q, -3, 0), D ** -0.5, cu_q=cu - 3)[:6])   # as many rows: the same split of the work
    assert (out[:3].view(torch.uint8) == MARK).all() and (out[9:].view(torch.uint8) == MARK).all() and untouched(raws)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_rows_take_the_codes_of_torchs_quantisers(cuda_device, fmt, dtype):
    """Scales and codes of unrotated rows are those that torch makes on the GPU, values between two codes among them.  E4M3 codes are
    compared as numbers: the kernel's division by correction makes +0 of -0 (fma(-q, s, x) is +0 there), the same value."""
    Hkv, D, T = 2, 128, 700
    table, total = page_table([15 if fmt == "pools" else 44], 0, torch.Generator().manual_seed(1))
    kv = empty_cache(fmt, total, Hkv, D, table, ints(0), 1, cuda_device)
    x = torch.randn(T, 2 * Hkv, D, generator=torch.Generator().manual_seed(2)) * torch.exp2(torch.arange(T) % 13 - 6.0)[:, None, None]
    x[::3] = (x[::3] * 4).round() / 4                # a coarse grid: many values lie between two codes
    x = x.to(dtype).to(cuda_device)
    paged.append_tokens(x.flatten(1), kv, 0, cu_new=offsets([T]).to(cuda_device))
    t = torch.arange(T, device=cuda_device)
    size = 48 if fmt == "pools" else 16
    page, slot = kv.page_table[0, t // size].long(), t % size
    held = lambda p: p.transpose(1, 2)[page, slot]  # noqa: E731
    for rows, which in ((x[:, :Hkv], "k"), (x[:, Hkv:], "v")):
        if fmt == "kv4":
            codes, scale = ds.quantize_groups_int4(rows)
            parts = paged.unpack_kv4(kv.buf)[:2] if which == "k" else paged.unpack_kv4(kv.buf)[2:]
        else:
            parts = (kv.k_pool, kv.k_scale) if which == "k" else (kv.v_pool, kv.v_scale)
            if fmt == "mixed" and which == "v":
                codes, scale = ds.quantize_rows_int4(rows)
            elif fmt in ("mixed", "e4m3"):
                codes, scale = ds.quantize_rows_e4m3(rows)
                codes, parts = codes.float(), (parts[0].float(), parts[1])
            else:
                amax = rows.float().abs().amax(-1)
                scale = torch.where(amax > 0, amax / 127.0, torch.ones_like(amax))
                codes = (rows.float() / scale[..., None]).round().to(torch.int8)
        assert torch.equal(held(parts[1]), scale) and torch.equal(held(parts[0]), codes)


@pytest.mark.parametrize("fmt", FORMATS)
def test_without_a_page_table(cuda_device, fmt):
    """Sequence b owns pages b * max_pages and on: the same bytes as with the table that says so."""
    size, per, B = (48 if fmt == "pools" else 16), 3, 3
    g = torch.Generator().manual_seed(8)
    lens, new = ints(0, size + 3, 2 * size + 1), [size + 5, 4, size]     # the last runs past its pages
    table = torch.arange(B * per, dtype=torch.int32).view(B, per)
    with_table, without = (empty_cache(fmt, B * per, 2, 128, table, lens, B, cuda_device) for _ in range(2))
    without.page_table = None
    qkv = torch.randn(sum(new), 7 * 128, generator=g).bfloat16().to(cuda_device)
    cu = offsets(new).to(cuda_device)
    q = [paged.append_tokens(qkv, kv, 3, cu_new=cu) for kv in (with_table, without)]
    assert torch.equal(*q) and all(torch.equal(a, b) for a, b in zip(cache_bytes(with_table), cache_bytes(without)))
    rows = [paged.read_tokens(kv, cu, sum(new), starts=kv.seq_lens) for kv in (with_table, without)]
    assert all(torch.equal(a, b) for a, b in zip(*rows)) and rows[0][0][-size:].any() and not rows[0][0][-1].any()


@pytest.mark.parametrize("fmt", ["kv4", "e4m3"])
def test_captured_with_offsets_made_in_the_graph(cuda_device, fmt):
    """Append and read-back captured with offsets and positions that the graph makes, replayed on changed inputs, an eager call on another
    stream meanwhile."""
    B, most = 40, 30
    table, total = page_table([3] * B, 0, torch.Generator().manual_seed(9))
    kv, other, plain = (empty_cache(fmt, total, 2, 128, table, ints(*range(B)), B, cuda_device) for _ in range(3))
    qkv = torch.zeros(B * most, 6 * 128, dtype=torch.float16, device=cuda_device)
    counts = torch.zeros(B, dtype=torch.int32, device=cuda_device)

    def work(cache):
        cu = torch.cat([counts[:1] * 0, counts.cumsum(0, dtype=torch.int32)])
        q = paged.append_tokens(qkv * 2, cache, 2, cu_new=cu + 0, q_out=torch.zeros(B * most, 2, 128, dtype=torch.float16, device=cuda_device))
        K, V = paged.read_tokens(cache, cu + 0, B * most, starts=cache.seq_lens + 0)
        here = torch.arange(B * most, device=cuda_device) < cu[-1]
        return q, torch.where(here[:, None, None], K, 0), torch.where(here[:, None, None], V, 0)

    work(kv)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = work(kv)
    side = torch.cuda.Stream()
    for seed in range(3):
        g = torch.Generator().manual_seed(seed)
        qkv.copy_(torch.randn(B * most, 6 * 128, generator=g))
        counts.copy_(torch.randint(0, most + 1 - 17, (B,), generator=g, dtype=torch.int32))
        torch.cuda.synchronize()
        graph.replay()
        with torch.cuda.stream(side):
            mixed = work(other)
        torch.cuda.synchronize()
        want = work(plain)
        assert all(torch.equal(a, b) for a, b in zip(got, want)) and all(torch.equal(a, b) for a, b in zip(mixed, want))
        assert all(torch.equal(a, b) for a, b in zip(cache_bytes(kv), cache_bytes(plain)))
