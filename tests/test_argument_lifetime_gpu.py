"""Tensors that a caller passes as temporaries (``cu_new=cu - first``) live until the kernel is launched: outputs and workspaces that a
call allocates must not be given their memory."""
import weakref

import pytest
import torch

from kv4_oracle import ints, offsets, page_table
from llm_inference_optimization_b200 import _lib, paged, rotary

pytestmark = pytest.mark.gpu


class Recorder:
    """Stands in for the library: notes which of the watched tensors are alive when an entry point is called."""

    def __init__(self):
        self.refs, self.alive, self.real = {}, {}, _lib.load()

    def temp(self, name, t):
        self.refs[name] = weakref.ref(t)
        return t

    def __getattr__(self, entry):
        if entry.endswith("workspace_bytes"):
            return getattr(self.real, entry)

        def call(*args):
            self.alive = {k: r() is not None for k, r in self.refs.items()}
            return 0
        return call


@pytest.mark.parametrize("what", ["append", "read", "decode", "rotary"])
def test_temporaries_live_until_the_launch(cuda_device, monkeypatch, what):
    dev = cuda_device
    table, total = page_table([2, 2], 0, torch.Generator().manual_seed(0))
    rec = Recorder()
    cache = lambda: paged.PagedKV4(torch.zeros(total, 2, 18, 64, dtype=torch.uint8, device=dev), rec.temp("table", table.to(dev)),  # noqa: E731
                                   rec.temp("lens", ints(4, 9).to(dev)), 2)
    rope = rotary.RotaryEmbedding(64, device=dev)
    monkeypatch.setattr(_lib, "load", lambda: rec)
    cu = lambda: rec.temp("cu", offsets([3, 2]).to(dev))  # noqa: E731
    status = lambda: rec.temp("status", torch.zeros(1, dtype=torch.int32, device=dev))  # noqa: E731
    if what == "append":
        paged.append_tokens(rec.temp("qkv", torch.zeros(5, 6 * 64, device=dev).half()), cache(), 2, rope, cu_new=cu(),
                            positions=rec.temp("positions", torch.arange(5, device=dev)), status=status())
    elif what == "read":
        paged.read_tokens(cache(), cu(), 5, starts=rec.temp("starts", ints(0, 1).to(dev)), status=status())
    elif what == "decode":
        cache().decode(rec.temp("q", torch.zeros(5, 4, 64, device=dev).half()), 0.125, cu_q=cu(), status=status())
    else:
        rope.apply(rec.temp("positions", torch.arange(5, device=dev)), rec.temp("q", torch.zeros(5, 2, 64, device=dev)),
                   rec.temp("k", torch.zeros(5, 1, 64, device=dev)))
    assert rec.alive and all(rec.alive.values()), rec.alive


def test_offsets_made_in_the_call(cuda_device):
    """More rows than one wave of blocks takes, offsets and positions made in the call: the rows that come last find them whole."""
    dev, B = cuda_device, 300
    new = [4 + i % 3 for i in range(B)]
    table, total = page_table([1] * B, 0, torch.Generator().manual_seed(1))
    zeros = ints(*[0] * B)
    cu, T = offsets(new).to(dev), sum(new)
    qkv = torch.randn(T, 6 * 128, generator=torch.Generator().manual_seed(2)).half().to(dev)
    kept, made = (paged.PagedKV4(torch.zeros(total, 2, 18, 128, dtype=torch.uint8, device=dev), table.to(dev), zeros.to(dev), B) for _ in range(2))
    want = paged.append_tokens(qkv, kept, 2, cu_new=cu)
    rows = paged.read_tokens(kept, cu, T)
    for _ in range(10):
        made.buf.zero_()
        got = paged.append_tokens(qkv, made, 2, cu_new=cu + 0)
        assert torch.equal(got, want) and torch.equal(made.buf, kept.buf)
        assert all(torch.equal(a, b) for a, b in zip(paged.read_tokens(made, cu + 0, T), rows))
        torch.cuda.empty_cache()
