"""4-bit attention at the limits of its arguments."""
import pytest
import torch

from kv4_oracle import ints, quantise4
from llm_inference_optimization_b200 import _C, paged

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("pages", [(1 << 28) + 1, 1 << 27])
def test_a_page_list_with_room_past_32_bits(cuda_device, pages):
    """Page lists of 2^28 + 1 and 2^27 entries have room for 2^32 + 16 and 2^31 tokens: the length decides what is read, and a
    largest length that 32 bits do not hold is refused."""
    g = torch.Generator().manual_seed(1)
    k, v = (quantise4(torch.randn(4, 2, 16, 64, generator=g)) for _ in range(2))
    buf = paged.pack_kv4(*k, *v).to(cuda_device)
    q, lens = torch.randn(1, 8, 64, generator=g).half().to(cuda_device), ints(57).to(cuda_device)
    want = _C.fused_gqa_kv4(q, buf, ints(2, 0, 3, 1).view(1, 4).to(cuda_device), lens, 0.125)
    table = torch.zeros(1, pages, dtype=torch.int32, device=cuda_device)
    table[0, :4] = ints(2, 0, 3, 1)
    assert torch.equal(_C.fused_gqa_kv4(q, buf, table, lens, 0.125), want)
    for longest in (2 ** 31 - 16, 2 ** 31, pages * 16 + 1):
        with pytest.raises(RuntimeError, match="max_seq_len"):
            _C.fused_gqa_kv4(q, buf, table, lens, 0.125, max_seq_len=longest)
    assert torch.equal(_C.fused_gqa_kv4(q, buf, table, lens, 0.125, max_seq_len=2 ** 31 - 17), want)
