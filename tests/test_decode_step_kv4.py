"""The decode step over caches of 4-bit keys and values, and with scaled rotary frequencies: host logic on the CPU, the
kernels' path on the GPU."""
import math

import pytest
import torch

from kv4_oracle import attend, offsets, values4
from llm_inference_optimization_b200 import decode_step as ds
from llm_inference_optimization_b200 import paged
from llm_inference_optimization_b200.sharding import shard_heads

LLAMA3 = {"type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0, "original_max_position": 8192}
CFG = ds.ModelConfig(layers=2, hidden=512, Hq=8, Hkv=2, D=128, mlp=1024, vocab=512, rope_scaling=LLAMA3)
LENS = torch.tensor([37, 5, 64], dtype=torch.int32)


def plain_attention(q, cache, page_table, seq_lens, scale, max_seq_len):
    """Attention over what a cache of 4-bit records holds, by the 64-bit formula."""
    k, ks, v, vs = (t.cpu() for t in paged.unpack_kv4(cache.buf))
    out = []
    for b in range(q.shape[0]):
        t = torch.arange(int(seq_lens[b]))
        row = lambda x: x.transpose(1, 2)[page_table[b].cpu()[t // 16].long(), t % 16]  # noqa: E731,B023
        o, _ = attend(q[b:b + 1].cpu().half(), values4(row(k), row(ks)), values4(row(v), row(vs)), row(vs).double().repeat_interleave(32, -1), scale, 1)
        out.append(o)
    return torch.cat(out).to(q.dtype).to(q.device)


def test_cpu_step_appends_and_attends():
    m = ds.DecodeModel(CFG, shard_heads(8, 2, 1, 0), "cpu", dtype=torch.float32, attention=plain_attention, v_bits=4, k_bits=4)
    m.init_cache(LENS)
    before = [paged.unpack_kv4(c.buf) for c in m.caches]
    logits = m.step(torch.tensor([3, 100, 250]))
    assert logits.shape == (3, 512) and torch.isfinite(logits).all() and torch.equal(m.seq_lens, LENS + 1)
    for c, old in zip(m.caches, before):                    # one token of every sequence changed, nothing else
        changed = torch.zeros(c.buf.shape[0], 16, dtype=torch.bool)
        for a, b in zip(old, paged.unpack_kv4(c.buf)):
            changed |= (a != b).any(-1).any(1)
        assert sorted(map(tuple, changed.nonzero().tolist())) == sorted((int(m.page_table[b, int(n) // 16]), int(n) % 16) for b, n in enumerate(LENS))


def test_scaled_frequencies_reach_the_plain_path():
    x, pos = torch.randn(3, 2, 128), torch.tensor([5, 4000, 100000])
    assert not torch.allclose(ds.rope(x, pos, 500000.0), ds.rope(x, pos, 500000.0, LLAMA3))
    assert torch.allclose(ds.rope(x, pos[:1].expand(3) * 0, 500000.0, LLAMA3), x)


def test_refusals():
    for bad in [dict(k_bits=4), dict(k_bits=2, v_bits=4), dict(k_bits=4, v_bits=4, layer_modes=["dense", "quest"]),
                dict(layer_modes=["quest", "quest"])]:
        with pytest.raises(ValueError):
            ds.DecodeModel(CFG, shard_heads(8, 2, 1, 0), "cpu", dtype=torch.float32, attention=plain_attention, **bad)
    m = ds.DecodeModel(CFG, shard_heads(8, 2, 1, 0), "cpu", dtype=torch.float32, attention=plain_attention, v_bits=4, k_bits=4)
    m.init_cache(LENS)
    with pytest.raises(RuntimeError):
        m.extend(torch.tensor([1, 2, 3]), offsets([1, 1, 1]))


def near(a, b, steps):
    """Relative distance in the 2-norm, in steps of bf16 rounding (2^-8 each)."""
    return float((a.float() - b.float()).norm() / b.float().norm()) <= steps * 2.0 ** -8


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [4, 8])
def test_kernel_path_matches_plain_path(cuda_device, bits):
    """The fused path (append_tokens, the attention kernels) against the torch path with the same bf16 weights.  Rows differ by
    the roundings of a dozen bf16 stages per layer, and by codes of the new token that such a difference turns."""
    kw = dict(dtype=torch.bfloat16, v_bits=4 if bits == 4 else 8, k_bits=bits)
    m = ds.DecodeModel(CFG, shard_heads(8, 2, 1, 0), cuda_device, **kw)
    plain = ds.DecodeModel(CFG, shard_heads(8, 2, 1, 0), cuda_device, attention=lambda *a: ds.kernel_attention(*a), **kw)
    assert m.fused_glue and not plain.fused_glue and m.rope is not None
    for x in (m, plain):
        x.init_cache(LENS)
    tok = torch.tensor([3, 100, 250], device=cuda_device)
    for _ in range(2):
        a, b = m.step(tok), plain.step(tok)
        assert near(a, b, 12)
        tok = b.argmax(-1)


@pytest.mark.gpu
def test_prompts_chunks_and_steps_agree(cuda_device):
    """A prompt taken whole, the same in chunks, and its last token as a step give the same logits, up to the roundings of
    matrix products of different shapes; the caches then hold the same tokens."""
    new = [40, 3, 90]
    g = torch.Generator().manual_seed(1)
    toks = [torch.randint(0, 512, (n,), generator=g) for n in new]
    whole, parts = (ds.DecodeModel(CFG, shard_heads(8, 2, 1, 0), cuda_device, dtype=torch.bfloat16, v_bits=4, k_bits=4) for _ in range(2))
    for m in (whole, parts):
        m.init_cache(torch.zeros(3, dtype=torch.int32), fill="zeros", extra_tokens=128)
    all_logits = whole.extend(torch.cat(toks).to(cuda_device), offsets(new).to(cuda_device))
    assert all_logits.shape == (sum(new), 512) and whole.seq_lens.tolist() == new
    first = [30, 0, 64]
    parts.extend(torch.cat([t[:n] for t, n in zip(toks, first)]).to(cuda_device), offsets(first).to(cuda_device))
    rest = [t[n:-1] for t, n in zip(toks, first)]
    parts.extend(torch.cat(rest).to(cuda_device), offsets([len(t) for t in rest]).to(cuda_device))
    last = parts.step(torch.stack([t[-1] for t in toks]).to(cuda_device))
    assert parts.seq_lens.tolist() == new
    ends = torch.tensor(new).cumsum(0) - 1
    assert near(last, all_logits[ends.to(cuda_device)], 12)
    # drafted tokens that are rejected are taken back by the lengths alone
    parts.extend(torch.tensor([1, 2, 3, 4, 5, 6], device=cuda_device), offsets([2, 2, 2]).to(cuda_device))
    parts.seq_lens.sub_(2)
    again = torch.tensor([7, 8, 9], device=cuda_device)
    assert near(parts.step(again), whole.step(again), 12)


@pytest.mark.gpu
def test_step_replays_from_a_graph(cuda_device):
    m = ds.DecodeModel(CFG, shard_heads(8, 2, 1, 0), cuda_device, dtype=torch.bfloat16, v_bits=4, k_bits=4)
    m.init_cache(LENS)
    tok = torch.tensor([3, 100, 250], device=cuda_device)
    m.step(tok)
    m.seq_lens.sub_(1)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = m.step(tok)
    m.seq_lens.copy_(LENS)
    graph.replay()
    got = out.clone()
    m.seq_lens.copy_(LENS)
    want = m.step(tok)
    torch.cuda.synchronize()
    assert torch.equal(got, want) and math.isfinite(float(got.float().sum()))


@pytest.mark.gpu
def test_padded_and_empty_prompts(cuda_device):
    """Tokens behind the last sequence change nothing for the others, in logits (up to roundings of matrix products of another
    shape) and lengths, nor is anything stored for a sequence without new ones; no tokens at all give no logits and leave the lengths."""
    toks = torch.randint(0, 512, (24,), generator=torch.Generator().manual_seed(2)).to(cuda_device)
    plain, padded = (ds.DecodeModel(CFG, shard_heads(8, 2, 1, 0), cuda_device, dtype=torch.bfloat16, v_bits=4, k_bits=4) for _ in range(2))
    for m in (plain, padded):
        m.init_cache(torch.zeros(3, dtype=torch.int32), fill="zeros", extra_tokens=64)
    cu = offsets([9, 0, 11]).to(cuda_device)
    a, b = plain.extend(toks[:20], cu), padded.extend(toks, cu)
    assert b.shape == (24, 512) and near(b[:20], a, 12)
    assert plain.seq_lens.tolist() == padded.seq_lens.tolist() == [9, 0, 11]
    untouched = padded.page_table[1].long()
    assert not any(c.buf[untouched].any() for c in padded.caches)
    none = padded.extend(toks[:0], offsets([0, 0, 0]).to(cuda_device))
    assert none.shape == (0, 512) and padded.seq_lens.tolist() == [9, 0, 11]


@pytest.mark.gpu
def test_prompt_replays_from_a_graph(cuda_device):
    m = ds.DecodeModel(CFG, shard_heads(8, 2, 1, 0), cuda_device, dtype=torch.bfloat16, v_bits=4, k_bits=4)
    m.init_cache(LENS, extra_tokens=64)
    toks = torch.randint(0, 512, (13,), generator=torch.Generator().manual_seed(3)).to(cuda_device)
    cu = offsets([4, 1, 8]).to(cuda_device)
    m.extend(toks, cu)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = m.extend(toks, cu)
    m.seq_lens.copy_(LENS)
    graph.replay()
    got = out.clone()
    m.seq_lens.copy_(LENS)
    want = m.extend(toks, cu)
    torch.cuda.synchronize()
    assert torch.equal(got, want)
