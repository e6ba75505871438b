"""Which destinations the rotation takes: rows that share memory are refused, others are not, whatever their strides."""
import itertools

import pytest
import torch

from llm_inference_optimization_b200 import _lib, rotary

NO_DEVICE = 9999     # the device is looked for behind the checks: a call that passes them ends there, before any launch


def verdict(lib, T, D, q, k=None, dtype=0):
    """q, k: (first element, heads, token stride, head stride) of views that are rotated in place; True where refused."""
    esz = 4 if dtype == 2 else 2
    at = [None if v is None else 4096 + v[0] * esz for v in (q, k)]
    heads = [0 if v is None else v[1] for v in (q, k)]
    st = [(0, 0) if v is None else v[2:] for v in (q, k)]
    rc = lib.skv_rotary(at[0], at[1], at[0], at[1], dtype, 16, 0, 16, T, heads[0], heads[1], D, D, 0, 1.0, 0, *st[0], *st[1], *st[0], *st[1],
                        NO_DEVICE, None)
    assert rc != 0 and (rc == -1) == ("overlap" in _lib.last_error()), _lib.last_error()
    return rc == -1


def shares(T, D, q, k=None):
    rows = [(o + t * a + h * b) for o, H, a, b in ([q] if k is None else [q, k]) for t in range(T) for h in range(H)]
    rows.sort()
    return any(y - x < D for x, y in zip(rows, rows[1:]))


@pytest.mark.parametrize("T,q,k", [(2, (0, 4, 128, 64), None),                       # a sliding window: rows (0,2) and (1,0) are one
                                   (3, (0, 4, 96, 64), None), (5, (0, 3, 64, 100), None),
                                   (4, (0, 5, 640, 64), (4 * 64, 4, 640, 64)),       # x[:, :5] and x[:, 4:8] of one projection
                                   (1, (0, 5, 640, 64), (4 * 64, 4, 640, 64)),
                                   (4, (0, 2, 640, 64), (32, 2, 640, 64)), (4, (0, 2, 256, 64), (256, 2, 512, 64))])
def test_views_that_share_rows_are_refused(lib, T, q, k):
    assert shares(T, 64, q, k) and verdict(lib, T, 64, q, k)


@pytest.mark.parametrize("T,q,k", [(7, (0, 5, 576, 64), (5 * 64, 2, 576, 64)),       # slices of a fused projection
                                   (7, (0, 3, 384, 128), (64, 3, 384, 128)),         # every other head
                                   (7, (0, 4, 64, 448), (4 * 448, 2, 64, 448)),      # heads outside, tokens inside
                                   (7, (0, 4, 64, 896), (448, 4, 64, 896)),
                                   (1, (0, 4, 0, 64), (256, 2, 0, 64)), (2, (0, 2, 128, 192), None),
                                   (4, (0, 2, 128, 64), (4096, 3, 192, 64))])
@pytest.mark.parametrize("dtype", [0, 2])
def test_views_that_do_not_are_taken(lib, T, q, k, dtype):
    assert not shares(T, 64, q, k) and not verdict(lib, T, 64, q, k, dtype)


def test_every_small_view(lib):
    """Against the rows themselves, all strides up to a few rows' lengths: one view, and two of one token stride."""
    D, wrong = 4, []
    for T, H, a, b in itertools.product((1, 2, 3, 5), (1, 2, 4), range(0, 26, 2), range(0, 26, 2)):
        if verdict(lib, T, D, (0, H, a, b)) != shares(T, D, (0, H, a, b)):
            wrong.append((T, H, a, b))
    for T, Hq, Hk, a, b, c, o in itertools.product((1, 2, 3), (1, 2), (1, 3), (0, 6, 12, 24), (4, 8, 10), (4, 12), range(-14, 30, 2)):
        q, k = (64, Hq, a, b), (64 + o, Hk, a, c)
        if verdict(lib, T, D, q, k) != shares(T, D, q, k):
            wrong.append((T, q, k))
    assert not wrong, (len(wrong), wrong[:5])


@pytest.mark.gpu
@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_unusual_views_in_place(cuda_device, layout):
    """Every other head, tokens inside heads: rotated in place they give what they give out of place."""
    r = rotary.RotaryEmbedding(64, layout=layout, device=cuda_device)
    pos = torch.arange(7, dtype=torch.int32, device=cuda_device) * 11
    base = torch.randn(7, 8, 64, generator=torch.Generator().manual_seed(1)).half().to(cuda_device)
    for view in (lambda x: (x[:, ::2], x[:, 1::2]), lambda x: (x[:, :5], x[:, 5:7]), lambda x: (x[:, 3:], x[:, :3])):
        for inside in (False, True):
            x = base.transpose(0, 1).contiguous().transpose(0, 1) if inside else base.clone()
            want = r.apply(pos, *view(x))
            got = r.apply(pos, *view(x), inplace=True)
            assert all(torch.equal(a, b) for a, b in zip(got, want))
    with pytest.raises(RuntimeError, match="overlap"):
        r.apply(pos, base[:, :5], base[:, 4:], inplace=True)
    with pytest.raises(RuntimeError, match="overlap"):
        r.apply(pos, base.view(56, 64).as_strided((7, 4, 64), (128, 64, 1)), inplace=True)
