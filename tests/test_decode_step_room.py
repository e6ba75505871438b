"""Decode models at the edges of their caches: prompts for part of a batch, sequences that outgrow their pages."""
import pytest
import torch

from kv4_oracle import offsets
from llm_inference_optimization_b200 import _workspace
from llm_inference_optimization_b200 import decode_step as ds
from llm_inference_optimization_b200.sharding import shard_heads
from test_decode_step_kv4 import CFG, near


@pytest.fixture
def clean_words(cuda_device):
    """The attention kernels report a missing page to their workspaces too, which later tests expect to be clean."""
    yield
    for kind in ("gqa", "gqa_kv4", "quest"):
        for ws in _workspace.all_of(kind, cuda_device):
            ws[:4].zero_()


KV4 = dict(dtype=torch.bfloat16, v_bits=4, k_bits=4)


def model(dev, lens, fill="zeros", extra=64, **kw):
    m = ds.DecodeModel(CFG, shard_heads(8, 2, 1, 0), dev, **kw)
    m.init_cache(torch.tensor(lens, dtype=torch.int32), fill=fill, extra_tokens=extra)
    return m


@pytest.mark.gpu
def test_prompt_whose_offsets_begin_above_zero(cuda_device):
    """Tokens before the first offset are padding, as those behind the last: what is cached stays, the others' logits too."""
    toks = torch.randint(0, 512, (24,), generator=torch.Generator().manual_seed(2)).to(cuda_device)
    whole, part = (model(cuda_device, [30, 5, 8], "normal", **KV4) for _ in range(2))
    before = [c.buf.clone() for c in part.caches]
    cu = offsets([9, 0, 11]).to(cuda_device)
    a, b = whole.extend(toks[4:], cu), part.extend(toks, cu + 4)
    assert near(b[4:], a, 12) and part.seq_lens.tolist() == whole.seq_lens.tolist() == [39, 5, 19]
    for c, old in zip(part.caches, before):                 # the tokens that were there: page 0 of sequence 0 whole, sequence 1
        page = int(part.page_table[0, 0])
        assert torch.equal(c.buf[page], old[page])
        own = part.page_table[1, :(5 + 64 + 15) // 16].long()
        assert torch.equal(c.buf[own], old[own])


def owned(m, b):
    """Pages of sequence b, by what init_cache gives it."""
    return m.page_table[b, :int(m.room[b]) // 16].long()


def test_entries_behind_a_sequences_pages_name_no_page():
    m = model("cpu", [500, 3], dtype=torch.float32, attention=lambda *a: None, v_bits=4, k_bits=4)
    assert m.room.tolist() == [(500 + 64 + 15) // 16 * 16, (3 + 64 + 15) // 16 * 16]
    pages = torch.cat([owned(m, 0), owned(m, 1)])
    assert sorted(pages.tolist()) == list(range(m.caches[0].buf.shape[0]))
    assert (m.page_table[1, int(m.room[1]) // 16:] == -1).all()
    m.check_cache()


@pytest.mark.parametrize("bits", [(8, 8), (8, 4), (4, 4)])
@pytest.mark.parametrize("lens", [(100, 80, 3), (176, 80, 80), (176, 40, 90), (176, 80, 3)])   # rooms 176, 80, 80
def test_plain_append_leaves_the_others_alone(bits, lens):
    """The torch append of a sequence at the end of its own pages, of the longest one too, and of all three at once."""
    m = model("cpu", [100, 10, 3], dtype=torch.float32, attention=lambda *a: None, k_bits=bits[0], v_bits=bits[1])
    assert m.room.tolist() == [176, 80, 80]
    cache = m.caches[0]
    cache.buf.copy_(torch.randint(0, 100, cache.buf.shape, generator=torch.Generator().manual_seed(1)))
    before = cache.buf.clone()
    k, v = (torch.randn(3, 2, 128, generator=torch.Generator().manual_seed(s)) for s in (2, 3))
    cache.append(k, v, m.page_table, torch.tensor(lens, dtype=torch.int32))
    single = ds.LayerCache(cache.buf.shape[0], 2, "cpu", bits[1], bits[0])
    single.buf.copy_(before)
    changed = []
    for b, n in enumerate(lens):                            # what each sequence with room does by itself
        if n < int(m.room[b]):
            single.append(k[b:b + 1], v[b:b + 1], m.page_table[b:b + 1], torch.tensor([n], dtype=torch.int32))
            changed.append(int(m.page_table[b, n // 16]))
    assert torch.equal(cache.buf, single.buf)
    assert sorted((cache.buf != before).flatten(1).any(1).nonzero().flatten().tolist()) == sorted(changed)


def test_check_cache_names_the_sequence():
    m = model("cpu", [100, 10, 3], dtype=torch.float32, attention=lambda *a: None)
    m.seq_lens[1] = 81
    with pytest.raises(RuntimeError, match=r"\[1\]"):
        m.check_cache()
    m.seq_lens[1] = 80
    m.check_cache()
    m.status.fill_(2)
    with pytest.raises(RuntimeError, match="status word 2"):
        m.check_cache()
    m.check_cache()


@pytest.mark.gpu
def test_a_prompt_past_a_sequences_own_pages(cuda_device, clean_words):
    """A short sequence beside a long one takes a prompt that its own pages do not hold: the long one's records stay, what fits
    is stored, and the model says so when asked."""
    m = model(cuda_device, [500, 3], "normal", **KV4)
    before = [c.buf.clone() for c in m.caches]
    toks = torch.randint(0, 512, (120,), generator=torch.Generator().manual_seed(5)).to(cuda_device)
    logits = m.extend(toks, offsets([0, 120]).to(cuda_device))
    assert logits.shape == (120, 512) and m.seq_lens.tolist() == [500, 123] and m.room.tolist() == [576, 80]
    for c, old in zip(m.caches, before):
        assert torch.equal(c.buf[owned(m, 0)], old[owned(m, 0)])
        assert not torch.equal(c.buf[owned(m, 1)[-1]], old[owned(m, 1)[-1]])
    with pytest.raises(RuntimeError, match=r"\[1\].*status word 2"):
        m.check_cache()


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [(8, 8), (8, 4), (4, 4)])
@pytest.mark.parametrize("fused", [True, False])
@pytest.mark.parametrize("scaled", [True, False])
def test_steps_past_a_sequences_own_pages(cuda_device, clean_words, bits, fused, scaled):
    cfg = CFG if scaled else ds.ModelConfig(layers=2, hidden=512, Hq=8, Hkv=2, D=128, mlp=1024, vocab=512)
    kw = {} if fused else dict(attention=lambda *a: ds.kernel_attention(*a))
    m = ds.DecodeModel(cfg, shard_heads(8, 2, 1, 0), cuda_device, dtype=torch.bfloat16, k_bits=bits[0], v_bits=bits[1], **kw)
    m.init_cache(torch.tensor([90, 3], dtype=torch.int32), extra_tokens=16)
    assert m.room.tolist() == [112, 32]
    before = [c.buf.clone() for c in m.caches]
    m.seq_lens.copy_(torch.tensor([90, 32]))
    tok = torch.tensor([3, 100], device=cuda_device)
    m.step(tok)
    for c, old in zip(m.caches, before):
        changed = (c.buf != old).flatten(1).any(1).nonzero().flatten().tolist()
        assert changed == [int(m.page_table[0, 90 // 16])]
    with pytest.raises(RuntimeError, match=r"\[1\]"):
        m.check_cache()
    m.seq_lens.copy_(torch.tensor([112, 31]))               # the longest at the table's own end
    before = [c.buf.clone() for c in m.caches]
    m.step(tok)
    for c, old in zip(m.caches, before):
        assert (c.buf != old).flatten(1).any(1).nonzero().flatten().tolist() == [int(m.page_table[1, 1])]
    with pytest.raises(RuntimeError, match=r"\[0\]"):
        m.check_cache()


@pytest.mark.gpu
def test_sparse_layers_allocate_no_dense_output(cuda_device, monkeypatch):
    """A block-sparse layer's attention brings its own output; a dense one's is allocated for it."""
    cfg = ds.ModelConfig(layers=2, hidden=512, Hq=8, Hkv=2, D=128, mlp=1024, vocab=512)
    m = ds.DecodeModel(cfg, shard_heads(8, 2, 1, 0), cuda_device, dtype=torch.bfloat16, layer_modes=["quest", "dense"])
    m.init_cache(torch.tensor([200, 90], dtype=torch.int32))
    made, real = [], torch.empty
    monkeypatch.setattr(ds.torch, "empty", lambda *a, **k: made.append((a[0], k.get("dtype"))) or real(*a, **k))
    for li in range(2):
        made.clear()
        qkv = torch.zeros(2, 12 * 128, dtype=torch.bfloat16, device=cuda_device)
        m._fused_attention(li, qkv, m.caches[li], m.seq_lens, m.seq_lens + 1, 0.1, torch.bfloat16)
        assert made.count(((2, 8, 128), torch.bfloat16)) == li


@pytest.mark.gpu
@pytest.mark.parametrize("v_bits", [8, 4])
def test_sparse_layers_past_a_sequences_own_pages(cuda_device, clean_words, v_bits):
    """A block-sparse layer beside a dense one: the sequence without room stores nothing, in its metadata neither."""
    cfg = ds.ModelConfig(layers=2, hidden=512, Hq=8, Hkv=2, D=128, mlp=1024, vocab=512)
    m = ds.DecodeModel(cfg, shard_heads(8, 2, 1, 0), cuda_device, dtype=torch.bfloat16, layer_modes=["quest", "dense"], v_bits=v_bits, quest_top_k=2)
    m.init_cache(torch.tensor([290, 30], dtype=torch.int32), extra_tokens=16)
    assert m.room.tolist() == [320, 48]
    m.seq_lens.copy_(torch.tensor([290, 48]))
    before, meta = [c.buf.clone() for c in m.caches], m.metas[0].clone()
    m.step(torch.tensor([3, 100], device=cuda_device))
    for c, old in zip(m.caches, before):
        assert (c.buf != old).flatten(1).any(1).nonzero().flatten().tolist() == [int(m.page_table[0, 290 // 16])]
    assert torch.equal(m.metas[0][1], meta[1])
    with pytest.raises(RuntimeError, match=r"\[1\]"):
        m.check_cache()
