"""4-bit page records and the argument checks of the append / read / 4-bit attention entry points, on the CPU."""
import pytest
import torch

from kv4_oracle import quantise4
from llm_inference_optimization_b200 import _lib, paged


@pytest.mark.parametrize("D", [64, 128])
def test_pack_and_unpack_are_inverse(D):
    g = torch.Generator().manual_seed(D)
    k, ks = quantise4(torch.randn(3, 2, 16, D, generator=g))
    v, vs = quantise4(torch.randn(3, 2, 16, D, generator=g))
    buf = paged.pack_kv4(k, ks, v, vs)
    assert buf.shape == (3, 2, 18, D) and buf.dtype == torch.uint8 and buf.is_contiguous()
    for a, b in zip(paged.unpack_kv4(buf), (k, ks, v, vs)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("D", [64, 128])
def test_bytes_lie_where_the_layout_says(D):
    g = torch.Generator().manual_seed(7)
    k, ks = quantise4(torch.randn(1, 1, 16, D, generator=g))
    v, vs = quantise4(torch.randn(1, 1, 16, D, generator=g))
    rec = paged.pack_kv4(k, ks, v, vs).flatten()
    nib = lambda at, n: (int(rec[at]) >> (4 * (n % 2))) % 16 - 8  # noqa: E731
    for t in range(16):
        i, j, e = t // 4, t // 2 % 2, t % 2
        place = 8 * j + 2 * i + e
        for d in range(D):
            w, c, n = d // 32, d % 32 // 8, d % 8
            assert nib(place * D // 2 + c * D // 8 + 4 * w + n // 2, n) == int(k[0, 0, t, d])
            gg, m = d % 32 // 4, d % 4
            assert nib(8 * D + j * 4 * D + gg * D // 2 + i * D // 8 + e * D // 16 + 2 * w + m // 2, m) == int(v[0, 0, t, d])
        sc = rec[16 * D + place * D // 8:16 * D + (place + 1) * D // 8].clone().view(torch.bfloat16)
        assert torch.equal(sc, torch.cat([ks[0, 0, t], vs[0, 0, t]]))


def test_wrong_shapes_are_refused():
    k, ks = torch.zeros(1, 1, 16, 64, dtype=torch.int8), torch.zeros(1, 1, 16, 2, dtype=torch.bfloat16)
    for args in [(k[:, :, :8], ks, k, ks), (k, ks.float(), k, ks), (k, ks[..., :1], k, ks), (k[..., :32], ks, k[..., :32], ks)]:
        with pytest.raises(RuntimeError):
            paged.pack_kv4(*args)
    with pytest.raises(RuntimeError):
        paged.unpack_kv4(torch.zeros(1, 1, 33, 128, dtype=torch.uint8))


def test_cache_object_and_cpu_refusal(lib):
    kv = paged.PagedKV4(torch.zeros(6, 2, 18, 64, dtype=torch.uint8), None, torch.zeros(2, dtype=torch.int32), 2)
    assert (kv.head_dim, kv.page_size, kv.max_pages, kv.capacity) == (64, 16, 3, 48)
    with pytest.raises(RuntimeError):
        kv.decode(torch.zeros(2, 4, 64, dtype=torch.float16), 0.125)
    with pytest.raises(RuntimeError):
        paged.append_tokens(torch.zeros(2, 8 * 64, dtype=torch.float16), kv, 4)
    with pytest.raises(RuntimeError):
        paged.read_tokens(kv, torch.zeros(3, dtype=torch.int32), 0)


def append_args(**kw):
    a = dict(qkv=16, bf16=0, stride=(4 + 4) * 64, q_out=16, q_bf16=0, freqs=None, R=0, inter=0, factor=1.0, pos=None, pos64=0, cu=None,
             table=None, lens=16, kp=16, vp=None, ks=None, vs=None, T=2, B=2, Hq=4, Hkv=2, D=64, fmt=_lib.KV_INT4, size=16, max_pages=3,
             pages=6, sp=2 * 18 * 64, sh=18 * 64, ss=0, csp=0, csh=0, status=None, dev=0, stream=None)
    assert set(kw) <= set(a)
    return list((a | kw).values())


@pytest.mark.parametrize("kw,code,word", [
    (dict(kp=None), -1, "null pool"), (dict(D=128, fmt=_lib.KV_E4M3), -1, "null pool"), (dict(fmt=_lib.KV_E4M3), -2, "head dim"),
    (dict(fmt=7), -2, "kv_dtype"), (dict(D=96), -2, "head dims"), (dict(size=32), -2, "16 tokens"), (dict(sh=1100), -1, "16 bytes"),
    (dict(kp=8), -1, "16 bytes"), (dict(qkv=8), -1, "16-byte"), (dict(stride=100), -1, "16-byte"), (dict(T=3), -1, "cu_new"),
    (dict(T=-1), -1, "sizes"), (dict(B=0, T=0), -1, "sizes"), (dict(pages=0), -1, "sizes"), (dict(qkv=None), -1, "null"),
    (dict(lens=None), -1, "null"), (dict(freqs=16, R=24), -2, "rotary_dim"), (dict(freqs=16, R=20, inter=1), -2, "rotary_dim"),
    (dict(freqs=16, R=80), -2, "rotary_dim"), (dict(fmt=_lib.KV_INT4 | 0x200), -2, "kv_dtype")])
def test_append_refuses(lib, kw, code, word):
    assert lib.skv_append_tokens(*append_args(**kw)) == code
    assert word in _lib.last_error()


def test_append_and_read_of_no_rows(lib):
    assert lib.skv_append_tokens(*append_args(T=0, cu=16, qkv=None)) == 0
    args = [16, None, None, None, None, 16, None, None, None, 0, 0, 2, 2, 64, _lib.KV_INT4, 16, 3, 6, 2304, 1152, 0, 0, 0, None, 0, None]
    assert lib.skv_read_tokens(*args) == 0
    args[10] = 4
    assert lib.skv_read_tokens(*args) == -1 and "null" in _lib.last_error()


def attend_args(**kw):
    a = dict(q=16, bf16=0, pool=16, table=None, lens=None, cu=None, out=16, out_bf16=0, ws=256, nbytes=1 << 30, T=2, B=2, N=48, Hq=4, Hkv=2,
             D=64, max_pages=3, pages=6, sp=2304, sh=1152, scale=0.125, status=None, dev=0, stream=None)
    assert set(kw) <= set(a)
    return list((a | kw).values())


@pytest.mark.parametrize("kw,code,word", [
    (dict(pool=None), -1, "null pool"), (dict(q=None), -1, "null"), (dict(Hq=5), -1, "divisible"), (dict(D=32), -2, "head dims"),
    (dict(N=49), -1, "max_pages"), (dict(T=3), -1, "cu_q"), (dict(scale=0.0), -1, "scale"), (dict(nbytes=100), -3, "workspace"),
    (dict(ws=None), -3, "workspace"), (dict(ws=272), -3, "aligned"), (dict(pool=8), -1, "16 bytes"), (dict(sp=2300), -1, "16 bytes"),
    (dict(q=8), -1, "16 bytes"), (dict(B=0), -1, "sizes"), (dict(Hkv=0), -1, "sizes"), (dict(sp=1 << 33), -2, "stride"),
    (dict(T=1 << 30, cu=16, Hq=16), -2, "rows")])
def test_attention_refuses(lib, kw, code, word):
    assert lib.skv_gqa_decode_kv4(*attend_args(**kw)) == code
    assert word in _lib.last_error()


def test_attention_of_no_rows_and_workspace_size(lib):
    assert lib.skv_gqa_decode_kv4(*attend_args(T=0, cu=16, q=None)) == 0
    assert lib.skv_gqa_decode_kv4_workspace_bytes(96) == 0
    assert 8192 < lib.skv_gqa_decode_kv4_workspace_bytes(64) < lib.skv_gqa_decode_kv4_workspace_bytes(128)
