"""Appending tokens to paged caches of every format and reading them back, against 64-bit plain forms."""
import pytest
import torch

from kv4_oracle import ints, offsets, page_table, quantise4, rotate, values4
from llm_inference_optimization_b200 import paged, rotary

pytestmark = pytest.mark.gpu
FORMATS = ["kv4", "e4m3", "int8", "mixed", "pools"]


def empty_cache(fmt, pages, Hkv, D, table, lens, B, dev, fill=0):
    if fmt == "kv4":
        return paged.PagedKV4(torch.full((pages, Hkv, 18, D), fill, dtype=torch.uint8, device=dev), table.to(dev), lens.to(dev), B)
    if fmt == "mixed":
        buf = torch.full((pages, Hkv, 25, 128), fill, dtype=torch.uint8, device=dev)
        return paged.PagedKV.from_mixed(buf, torch.float8_e4m3fn, table.to(dev), lens.to(dev), B)
    if fmt == "pools":   # separate pools of 48-token pages
        mk = lambda dt, *s: torch.zeros((pages, Hkv, 48, *s), dtype=dt, device=dev)  # noqa: E731
        return paged.PagedKV(mk(torch.int8, 128), mk(torch.int8, 128), mk(torch.float32), mk(torch.float32), table.to(dev), lens.to(dev), B)
    code = torch.int8 if fmt == "int8" else torch.float8_e4m3fn
    buf = torch.full((pages, Hkv, 33, 128), fill, dtype=torch.uint8, device=dev)
    return paged.PagedKV.from_fused(buf, code, table.to(dev), lens.to(dev), B)


def rows_of(kv, table, b, pos):
    """What the cache holds for positions `pos` of sequence b: codes and scales as 64-bit numbers, per channel."""
    size = 16 if isinstance(kv, paged.PagedKV4) else kv.page_size
    page, slot = table[b, pos // size].long(), pos % size
    if isinstance(kv, paged.PagedKV4):
        k, ks, v, vs = (t.cpu() for t in paged.unpack_kv4(kv.buf))
        wide = lambda s: s.double().repeat_interleave(32, -1)  # noqa: E731
    else:
        k, ks, v, vs = kv.k_pool.cpu().float(), kv.k_scale.cpu(), kv.v_pool.cpu(), kv.v_scale.cpu()
        if kv.v_bits == 4:
            v = torch.stack([v & 15, v >> 4], -1).flatten(-2).to(torch.int8) - 8
        else:
            v = v.float()
        wide = lambda s: s.double()[..., None].expand(*s.shape, 128)  # noqa: E731
    at = lambda t: t.transpose(1, 2)[page, slot]  # noqa: E731        [n, Hkv, ...]
    return at(k).double(), at(wide(ks)), at(v).double(), at(wide(vs))


def check_held(x, codes, scale, kind):
    """x (64-bit) is held as codes * scale: the scale is amax / top, rounded; the value within half a step of x."""
    top = {"kv4": 7.0, "int4": 7.0, "int8": 127.0, "e4m3": 448.0}[kind]
    group = 32 if kind == "kv4" else 128
    amax = x.unflatten(-1, (-1, group)).abs().amax(-1).repeat_interleave(group, -1)
    want = amax / top
    # bf16 scale: half a step (2^-8); fp32: a division and the 32-bit rotation (1e-6 of the largest pair)
    assert ((scale - want).abs() <= want * (2.0 ** -8 if kind == "kv4" else 2.0 ** -23) + 2e-6 * want + (want == 0) * 1.0).all()
    off = (codes * scale - x).abs()
    if kind == "e4m3":     # half a step of 3 bits behind the leading one, 2^-10 below the smallest normal
        tol = torch.maximum(x.abs() * 2.0 ** -4, scale * 2.0 ** -10)
    else:
        tol = scale * 0.5
    # the rotated value is off by 1e-6 of its pair, at most twice the group's... the largest of the row
    slack = x.abs().amax(-1, keepdim=True) * 3e-6
    assert (off <= tol * (1 + 1e-6) + slack).all(), float((off / (tol + slack + 1e-300)).max())


def run_case(fmt, old, new, Hq, Hkv, D, dev, *, dtype=torch.bfloat16, layout="half", R=None, seed=0, scaling=None, positions=None,
             cu_none=False, pad_rows=0, strided=False, rope=True):
    g = torch.Generator().manual_seed(seed)
    B, T = len(new), sum(new)
    size = 48 if fmt == "pools" else 16
    table, total = page_table([(a + n + size - 1) // size + 1 for a, n in zip(old, new)], 3, g)
    kv = empty_cache(fmt, total, Hkv, D, table, ints(*old), B, dev)
    x = torch.randn(T + pad_rows, Hq + 2 * Hkv, D, generator=g)
    x[..., :2] *= 8
    if T:
        x[0, Hq + Hkv] = 0                           # a value row of zeros
        x[0, -1, D // 2:] *= 2.0 ** -30              # and one with a tiny half
    x = x.to(dtype)
    qkv = x.flatten(1).to(dev)
    if strided:
        wide = torch.zeros(T + pad_rows, qkv.shape[1] + 64, dtype=dtype, device=dev)
        wide[:, :qkv.shape[1]] = qkv
        qkv = wide[:, :qkv.shape[1]]
    r = rotary.RotaryEmbedding(D, 500000.0, rotary_dim=R, layout=layout, scaling=scaling, device=dev) if rope else None
    q_out = torch.full((T + pad_rows, Hq, D), 77.0, dtype=torch.float16, device=dev)
    st = torch.zeros(1, dtype=torch.int32, device=dev)
    q = paged.append_tokens(qkv, kv, Hq, r, cu_new=None if cu_none else offsets(new).to(dev), q_out=q_out, status=st,
                            positions=None if positions is None else positions.to(dev))
    assert q is q_out and int(st) == 0
    place = torch.cat([torch.arange(a, a + n) for a, n in zip(old, new)]) if T else torch.zeros(0, dtype=torch.long)
    if rope:
        f, a = rotary.frequencies(r.rotary_dim, 500000.0, scaling)
        turned = rotate(x[:T, :Hq + Hkv], place if positions is None else positions[:T], f, a, layout)
    else:
        turned = x[:T, :Hq + Hkv].double()
    want_q = turned[:, :Hq]
    tol = want_q.abs() * 2.0 ** -11 + 2.0 ** -25 + x[:T].double().abs().amax() * 4e-6
    assert ((q[:T].double().cpu() - want_q).abs() <= tol).all()
    assert (q[T:] == 77.0).all()
    at = 0
    for b, n in enumerate(new):
        if n:
            kc, ks, vc, vs = rows_of(kv, table, b, torch.arange(old[b], old[b] + n))
            key = {"kv4": "kv4", "e4m3": "e4m3", "int8": "int8", "mixed": "e4m3", "pools": "int8"}[fmt]
            check_held(turned[at:at + n, Hq:], kc, ks, key)
            v = x[at:at + n, Hq + Hkv:]
            check_held(v.double(), vc, vs, "int4" if fmt == "mixed" else key)
            if fmt == "kv4":                         # unrotated rows: the codes and scales of 32-bit arithmetic, bit for bit
                c, s = quantise4(v)
                assert torch.equal(c.double(), vc) and torch.equal(s.double().repeat_interleave(32, -1), vs)
            at += n
    return kv, table, x


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("old,new", [([0], [1]), ([5, 0, 16, 31], [1, 1, 1, 1]), ([0, 250, 33], [65, 17, 130]), ([3, 0, 7], [0, 40, 0])])
def test_append_every_format(cuda_device, fmt, old, new):
    run_case(fmt, old, new, 8, 2, 128, cuda_device, seed=len(old))


@pytest.mark.parametrize("layout,R", [("half", 64), ("half", 16), ("half", 48), ("interleaved", 64), ("interleaved", 8), ("interleaved", 40)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_append_narrow_heads_and_partial_rotation(cuda_device, layout, R, dtype):
    run_case("kv4", [9, 100], [21, 6], 3, 1, 64, cuda_device, dtype=dtype, layout=layout, R=R, seed=R)
    run_case("kv4", [9, 100], [21, 6], 5, 5, 128, cuda_device, dtype=dtype, layout=layout, R=R, seed=R + 1)


def test_append_one_row_each_without_offsets(cuda_device):
    run_case("kv4", [0, 15, 16, 1000, 7], [1] * 5, 32, 8, 128, cuda_device, cu_none=True)
    run_case("int8", [0, 15, 16], [1] * 3, 4, 4, 128, cuda_device, cu_none=True, rope=False)


@pytest.mark.parametrize("B", [200, 300])            # counted by all lanes of a row; searched
def test_append_many_sequences_some_empty(cuda_device, B):
    new = [(i * 7) % 4 for i in range(B)]
    run_case("kv4", [i % 40 for i in range(B)], new, 4, 2, 64, cuda_device, seed=B, scaling={"type": "linear", "factor": 4.0})


def test_rows_behind_the_last_sequence_are_left_alone(cuda_device):
    run_case("kv4", [4, 0], [5, 9], 4, 2, 128, cuda_device, pad_rows=6, strided=True)
    run_case("e4m3", [4, 0], [5, 9], 4, 2, 128, cuda_device, pad_rows=1, strided=True)


@pytest.mark.parametrize("dt", [torch.int32, torch.int64])
def test_positions_may_differ_from_places(cuda_device, dt):
    pos = torch.tensor([100000, 7, 8, 1 << 20, 5, 6, 7, 0, 0], dtype=dt)
    run_case("kv4", [4, 30], [4, 5], 4, 2, 128, cuda_device, positions=pos)


@pytest.mark.parametrize("fmt", FORMATS)
def test_tokens_before_are_left_and_old_ones_overwritten(cuda_device, fmt):
    """A second append touches its own tokens only, also inside a shared page and byte-neighbouring tokens."""
    kv, table, _ = run_case(fmt, [0, 0], [37, 5], 2, 2, 128, cuda_device, seed=3)
    before = rows_of(kv, table, 0, torch.arange(37)), rows_of(kv, table, 1, torch.arange(5))
    kv.seq_lens.copy_(ints(33, 5))
    g = torch.Generator().manual_seed(5)
    qkv = torch.randn(3, 6 * 128, generator=g).half().to(cuda_device)
    paged.append_tokens(qkv, kv, 2, cu_new=offsets([2, 1]).to(cuda_device))
    for b, keep in ((0, [*range(33), 35, 36]), (1, [*range(5)])):
        for x, y in zip(before[b], rows_of(kv, table, b, torch.tensor(keep))):
            assert torch.equal(x[keep], y)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_read_returns_what_is_held(cuda_device, fmt, dtype):
    kv, table, _ = run_case(fmt, [0, 0, 0], [37, 16, 70], 2, 3, 128, cuda_device, seed=4)
    counts, starts = [20, 0, 64], [17, 3, 2]
    K, V = paged.read_tokens(kv, offsets(counts).to(cuda_device), 84 + 2, starts=ints(*starts).to(cuda_device), dtype=dtype)
    at = 0
    for b, n in enumerate(counts):
        kc, ks, vc, vs = rows_of(kv, table, b, torch.arange(starts[b], starts[b] + n))
        assert torch.equal(K[at:at + n].cpu(), (kc.float() * ks.float()).to(dtype))
        assert torch.equal(V[at:at + n].cpu(), (vc.float() * vs.float()).to(dtype))
        at += n
    K0, _ = paged.read_tokens(kv, offsets([37, 16, 70]).to(cuda_device), 123, dtype=dtype)
    assert torch.equal(K0[17:37], K[:20])


@pytest.mark.parametrize("fmt", FORMATS)
def test_rows_that_are_not_finite_say_so(cuda_device, fmt):
    B, Hkv = 3, 2
    table, total = page_table([2, 2, 2], 0, torch.Generator().manual_seed(0))
    kv = empty_cache(fmt, total, Hkv, 128, table, ints(0, 3, 16), B, cuda_device)
    x = torch.randn(3, 2 * Hkv, 128, generator=torch.Generator().manual_seed(1))
    x[0, 0, 5] = float("nan")
    x[1, 3, 127] = float("inf")
    paged.append_tokens(x.flatten(1).half().to(cuda_device), kv, 0)
    K, V = paged.read_tokens(kv, offsets([1, 1, 1]).to(cuda_device), 3, starts=ints(0, 3, 16).to(cuda_device))
    wide = 32 if fmt == "kv4" else 128
    bad_k = torch.zeros(3, Hkv, 128, dtype=torch.bool)
    bad_v = bad_k.clone()
    bad_k[0, 0, :wide] = True
    bad_v[1, 1, 128 - wide:] = True
    assert torch.equal(torch.isnan(K).cpu(), bad_k) and torch.equal(torch.isnan(V).cpu(), bad_v)


@pytest.mark.parametrize("fmt", ["kv4", "e4m3"])
@pytest.mark.parametrize("bad", [-1, 1 << 20, 2 ** 31 - 1])
def test_bad_pages_and_full_sequences_store_nothing(cuda_device, fmt, bad):
    table, total = page_table([2, 2], 1, torch.Generator().manual_seed(2))
    table[1, 0] = bad
    kv = empty_cache(fmt, total, 2, 128, table, ints(30, 0), 2, cuda_device)
    buf = kv.buf if fmt == "kv4" else kv.k_pool
    qkv = torch.randn(10, 6 * 128, generator=torch.Generator().manual_seed(3)).half().to(cuda_device)
    st = torch.zeros(1, dtype=torch.int32, device=cuda_device)
    q = paged.append_tokens(qkv, kv, 2, cu_new=offsets([6, 4]).to(cuda_device), status=st)   # 30, 31 fit, the rest does not
    assert int(st) == 2 and torch.equal(q.flatten(1), qkv[:, :256])
    touched = buf.view(torch.uint8).flatten(1).any(1).nonzero().flatten().tolist()
    assert touched == [int(table[0, 1])]
    st.zero_()
    K, V = paged.read_tokens(kv, offsets([6, 4]).to(cuda_device), 10, starts=ints(30, 0).to(cuda_device), status=st)
    assert int(st) == 2 and (K[2:] == 0).all() and (V[2:] == 0).all() and (K[:2] != 0).any()
    # negative places are no places
    kv.seq_lens.copy_(ints(-3, -3))
    buf.view(torch.uint8).zero_()
    paged.append_tokens(qkv[:2], kv, 2, cu_new=offsets([2, 0]).to(cuda_device))
    assert not buf.view(torch.uint8).any()


def test_offsets_that_do_not_ascend_stay_in_bounds(cuda_device):
    table, total = page_table([3, 3, 3], 0, torch.Generator().manual_seed(4))
    kv = empty_cache("kv4", total, 2, 64, table, ints(0, 0, 0), 3, cuda_device)
    guard = torch.zeros_like(kv.buf)
    qkv = torch.randn(9, 6 * 64, generator=torch.Generator().manual_seed(3)).half().to(cuda_device)
    for cu in [(5, 2, 9, 1), (-7, 100, -100, 3), (2 ** 31 - 1, -2 ** 31, 0, 9)]:
        paged.append_tokens(qkv, kv, 2, cu_new=ints(*cu).to(cuda_device))
        paged.read_tokens(kv, ints(*cu).to(cuda_device), 9)
        kv.decode(torch.randn(9, 2, 64, device=cuda_device).half(), 0.125, cu_q=ints(*cu).to(cuda_device))
    torch.cuda.synchronize()
    assert not guard.any()


def test_one_layer_of_an_interleaved_buffer(cuda_device):
    """A view with strided pages: [pages, layers, Hkv, 18, D][:, 1]."""
    g = torch.Generator().manual_seed(6)
    table, total = page_table([4], 0, g)
    big = torch.zeros(total, 3, 2, 18, 64, dtype=torch.uint8, device=cuda_device)
    kv = paged.PagedKV4(big[:, 1], table.to(cuda_device), ints(0).to(cuda_device), 1)
    qkv = torch.randn(50, 4 * 64, generator=g).half().to(cuda_device)
    paged.append_tokens(qkv, kv, 0, cu_new=offsets([50]).to(cuda_device))
    assert not big[:, 0].any() and not big[:, 2].any()
    K, V = paged.read_tokens(kv, offsets([50]).to(cuda_device), 50)
    x = qkv.cpu().view(50, 4, 64)
    for got, rows in ((K, x[:, :2]), (V, x[:, 2:])):
        c, s = quantise4(rows)
        assert torch.equal(got.cpu(), values4(c, s).half())


def test_refusals(cuda_device):
    table, total = page_table([2, 2], 0, torch.Generator().manual_seed(0))
    kv = empty_cache("kv4", total, 2, 64, table, ints(0, 0), 2, cuda_device)
    qkv = torch.zeros(2, 8 * 64, dtype=torch.float16, device=cuda_device)
    r128 = rotary.RotaryEmbedding(128, device=cuda_device)
    odd = rotary.RotaryEmbedding(64, rotary_dim=24, device=cuda_device)
    no_lens = paged.PagedKV4(kv.buf, kv.page_table, None, 2)
    wrong = paged.PagedKV4(kv.buf[..., :32], kv.page_table, kv.seq_lens, 2)
    for bad in [lambda: paged.append_tokens(qkv, kv, 4, r128), lambda: paged.append_tokens(qkv, kv, 4, odd), lambda: paged.append_tokens(qkv, kv, 5),
                lambda: paged.append_tokens(qkv[:1], kv, 4), lambda: paged.append_tokens(qkv.float(), kv, 4),
                lambda: paged.append_tokens(qkv, no_lens, 4), lambda: paged.append_tokens(qkv, wrong, 4),
                lambda: paged.append_tokens(qkv, kv, 4, cu_new=torch.zeros(3, dtype=torch.int64, device=cuda_device)),
                lambda: paged.append_tokens(qkv, kv, 4, positions=torch.zeros(3, dtype=torch.int32, device=cuda_device)),
                lambda: paged.append_tokens(qkv, kv, 4, q_out=torch.zeros(2, 4, 64, device=cuda_device)),
                lambda: paged.append_tokens(qkv[:, 4:], kv, 4), lambda: paged.append_tokens(qkv.cpu(), kv, 4),
                lambda: paged.read_tokens(kv, ints(0, 1, 2), 2), lambda: paged.read_tokens(kv, ints(0, 1, 2).to(cuda_device), -1),
                lambda: paged.read_tokens(kv, ints(0, 1, 2).to(cuda_device), 2, dtype=torch.float32)]:
        with pytest.raises(RuntimeError):
            bad()
