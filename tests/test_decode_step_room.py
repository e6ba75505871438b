"""Decode models at the edges of their caches: prompts for part of a batch, sequences that outgrow their pages."""
import pytest
import torch

from kv4_oracle import offsets
from llm_inference_optimization_b200 import decode_step as ds
from llm_inference_optimization_b200.sharding import shard_heads
from test_decode_step_kv4 import CFG, near

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
