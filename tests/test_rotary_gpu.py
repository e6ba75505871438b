"""The rotation kernel against the 64-bit formula: layouts, widths, types, strides, far positions, gradients."""
import pytest
import torch

from kv4_oracle import close, half_step, rotate, rotate_slack
from llm_inference_optimization_b200 import rotary

pytestmark = pytest.mark.gpu
LLAMA3 = {"type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0, "original_max_position": 8192}
YARN = {"type": "yarn", "factor": 16.0, "original_max_position": 4096}


def rows(shape, dtype, seed):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


def check(r, x, pos, got, adjoint=False, theta=10000.0, scaling=None):
    f, a = rotary.frequencies(r.rotary_dim, theta, scaling)
    want = rotate(x, pos, f, a, r.layout, adjoint)
    close(got, want, half_step(want, x.dtype) + rotate_slack(x, r.layout, r.rotary_dim, a))
    assert torch.equal(got[..., r.rotary_dim:].cpu(), x[..., r.rotary_dim:])


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T,Hq,Hk,D,R", [(1, 1, 1, 64, 64), (3, 8, 2, 128, 128), (17, 4, 1, 128, 64), (5, 3, 3, 96, 96), (257, 2, 1, 80, 20),
                                         (2, 5, 1, 64, 2), (9, 7, 1, 160, 30), (33, 1, 1, 256, 256), (7, 3, 2, 66, 22), (4, 2, 1, 63, 6)])
def test_matches_formula(cuda_device, layout, dtype, T, Hq, Hk, D, R):
    r = rotary.RotaryEmbedding(D, rotary_dim=R, layout=layout, device=cuda_device)
    q, k = rows((T, Hq, D), dtype, 1), rows((T, Hk, D), dtype, 2)
    pos = torch.randint(0, 5000, (T,), generator=torch.Generator().manual_seed(3), dtype=torch.int32)
    qo, ko = r.apply(pos.to(cuda_device), q.to(cuda_device), k.to(cuda_device))
    check(r, q, pos, qo)
    check(r, k, pos, ko)


@pytest.mark.parametrize("scaling", [None, LLAMA3, YARN, {"type": "ntk", "factor": 4.0}, {"type": "linear", "factor": 4.0}])
@pytest.mark.parametrize("pos64", [False, True])
def test_far_positions_keep_their_angles(cuda_device, scaling, pos64):
    """A 32-bit angle is off by tenths of a radian at these positions; the tolerance is that of position 1."""
    r = rotary.RotaryEmbedding(128, 500000.0, scaling=scaling, device=cuda_device)
    pos = [0, 1, 131071, 1 << 20, (1 << 24) + 1, (1 << 31) - 1] + ([1 << 33, -5] if pos64 else [-1])
    pos = torch.tensor(pos, dtype=torch.int64 if pos64 else torch.int32)
    x = rows((len(pos), 2, 128), torch.float32, 4)
    # frequencies carry 2^-53 of relative rounding, in the oracle as in the kernel: 2^33 * 2^-52 radians at most
    f, a = rotary.frequencies(128, 500000.0, scaling)
    want = rotate(x, pos, f, a, "half")
    got = r.apply(pos.to(cuda_device), x.to(cuda_device))
    close(got, want, half_step(want, torch.float32) + rotate_slack(x, "half", 128, a) * (1 + 4))


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_gradient_matches_formula_and_differences(cuda_device, layout, dtype):
    r = rotary.RotaryEmbedding(64, rotary_dim=48, layout=layout, scaling=YARN, device=cuda_device)
    pos = torch.tensor([0, 7, 1000, 60001], dtype=torch.int32)
    g = rows((4, 3, 64), dtype, 5)
    got = r.apply(pos.to(cuda_device), g.to(cuda_device), adjoint=True)
    check(r, g, pos, got, adjoint=True, scaling=YARN)
    # <g, J e> by differences of the (linear) map: J e = apply(x + e) - apply(x), for a few channels
    if dtype == torch.float32:
        x = rows((4, 3, 64), dtype, 6)
        f, a = rotary.frequencies(48, 10000.0, YARN)
        for c in (0, 1, 23, 24, 47, 63):
            e = torch.zeros_like(x)
            e[..., c] = 0.5
            moved = r.apply(pos.to(cuda_device), (x + e).to(cuda_device)).cpu().double() - r.apply(pos.to(cuda_device), x.to(cuda_device)).cpu().double()
            want = (moved * g.double()).sum(-1) / 0.5
            tol = 64 * 2.0 ** -22 * a * 8          # differences of 32-bit values of a few units, summed over 64 channels
            assert (got[..., c].cpu().double() - want).abs().max().item() <= tol


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_strided_views_and_in_place(cuda_device, dtype):
    r = rotary.RotaryEmbedding(64, rotary_dim=32, device=cuda_device)
    both = rows((11, 9, 64), dtype, 7)
    pos = torch.arange(11, dtype=torch.int32) * 3
    d = both.to(cuda_device)
    q, k = d[:, :6], d[:, 6:8]                       # the ninth head is a value head and stays
    qo, ko = r.apply(pos.to(cuda_device), q, k)
    assert qo.is_contiguous() and ko.is_contiguous() and torch.equal(d.cpu(), both)
    check(r, both[:, :6], pos, qo)
    back = r.apply(pos.to(cuda_device), q, k, inplace=True)
    assert back[0].data_ptr() == q.data_ptr()
    assert torch.equal(d[:, :6], qo) and torch.equal(d[:, 6:8], ko) and torch.equal(d[:, 8].cpu(), both[:, 8])
    odd = torch.empty(11 * 6 * 67 + 1, dtype=dtype, device=cuda_device)[1:].view(11, 6, 67)[..., :64]   # rows on no wide boundary
    odd.copy_(both[:, :6])
    assert torch.equal(r.apply(pos.to(cuda_device), odd), qo)


def test_only_rotates_and_turns_back(cuda_device):
    """Norms of pairs stay; the gradient's map is the inverse where the factor is one."""
    r = rotary.RotaryEmbedding(128, device=cuda_device)
    x = rows((300, 8, 128), torch.float32, 8).to(cuda_device)
    pos = torch.arange(300, dtype=torch.int64, device=cuda_device) * 1001
    y = r.apply(pos, r.apply(pos, x), adjoint=True)
    assert (y - x).abs().max().item() <= 5e-6 * x.abs().max().item()


def test_no_rows_other_streams_and_graphs(cuda_device):
    r = rotary.RotaryEmbedding(64, device=cuda_device)
    assert r.apply(torch.empty(0, dtype=torch.int32, device=cuda_device), torch.empty(0, 4, 64, device=cuda_device)).shape == (0, 4, 64)
    x, pos = rows((5, 4, 64), torch.float16, 9).to(cuda_device), torch.arange(5, dtype=torch.int32, device=cuda_device)
    want = r.apply(pos, x)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = r.apply(pos, x)
    s.synchronize()
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = r.apply(pos, x)
    x.mul_(2)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, r.apply(pos, x))


def test_refusals(cuda_device):
    r = rotary.RotaryEmbedding(64, device=cuda_device)
    x, pos = torch.zeros(3, 2, 64, device=cuda_device), torch.zeros(3, dtype=torch.int32, device=cuda_device)
    for bad in [lambda: r.apply(pos[:2], x), lambda: r.apply(pos.float(), x), lambda: r.apply(pos, x.double()),
                lambda: r.apply(pos, x[..., :32]), lambda: r.apply(pos, x, x.half()), lambda: r.apply(pos.cpu(), x),
                lambda: r.apply(pos, x.transpose(1, 2).contiguous().transpose(1, 2)), lambda: r.apply(pos, x, x[:2]),
                lambda: r.apply(pos, x.clone().requires_grad_()),
                lambda: rotary.RotaryEmbedding(64, device="cpu").apply(pos, x)]:
        with pytest.raises(RuntimeError):
            bad()
