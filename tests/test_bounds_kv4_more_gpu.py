"""The range-checking library over the wider run of rotation, append, read-back and 4-bit attention: every layout and width, searched
and unusual offsets, many sequences, items that span blocks, page tables with entries outside the pool.  Positions in page tables,
offsets and lengths, rows, heads, channels, angle tables, ring and partial-result places are checked in that build.  It is
chosen per process, so the driver runs in a child process; it prints one JSON line."""
import json
import os
import subprocess
import sys
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]
pytestmark = pytest.mark.gpu

DRIVER = r'''
import ctypes as C, itertools, json, sys
import torch
sys.path[:0] = [%(root)r, %(root)r + "/tests"]
from kv4_oracle import half_step, ints, offsets, page_table, quantise4, rotate, rotate_slack
from test_kv_tokens_gpu import FORMATS, empty_cache
from llm_inference_optimization_b200 import _lib, paged, rotary
lib = _lib.load()
dev = torch.device("cuda", 0)
g = torch.Generator().manual_seed(1)
raws, seen, ok = [], {}, {}

def canary(shape, dtype):
    n = int(torch.tensor(shape).prod()) * torch.empty((), dtype=dtype).element_size()
    raw = torch.full((n + 8192,), 0xA5, dtype=torch.uint8, device=dev)
    raws.append(raw)
    return raw[4096:4096 + n].view(dtype).view(shape)

def done(name):
    """Violations so far, and whether the guard bytes of this part stand."""
    torch.cuda.synchronize()
    for f in ("kv_tokens", "gqa_decode_kv4", "rotary"):
        get = getattr(lib, "skv_debug_bounds_" + f)
        get.restype, get.argtypes = C.c_int, [C.POINTER(C.c_int)]
        v = C.c_int(-1)
        assert get(C.byref(v)) == 0
        if v.value:
            seen.setdefault(f, (name, v.value))
    ok[name] = all(bool((r[:4096] == 0xA5).all() and (r[-4096:] == 0xA5).all()) for r in raws)
    raws.clear()

good = True
for (T, Hq, Hk, D, R), layout, dtype in itertools.product(
        [(1, 1, 1, 64, 64), (17, 4, 1, 128, 64), (5, 3, 3, 96, 96), (257, 2, 1, 80, 20), (2, 5, 1, 64, 2), (9, 7, 1, 160, 30), (7, 3, 2, 66, 22),
         (4, 2, 1, 63, 6), (3, 70, 2, 256, 256), (2, 1, 1, 4096, 1030)], ["half", "interleaved"], [torch.float16, torch.float32]):
    r = rotary.RotaryEmbedding(D, rotary_dim=R, layout=layout, device=dev)
    x = torch.randn(T, Hq + Hk, D, generator=g).to(dtype)
    both = canary((T, Hq + Hk, D), dtype)
    both.copy_(x)
    pos = torch.randint(0, 5000, (T,), generator=g, dtype=torch.int32)
    out = r.apply(pos.to(dev), both[:, :Hq], both[:, Hq:])
    r.apply(pos.to(dev), both[:, :Hq], both[:, Hq:], inplace=True)
    good &= torch.equal(torch.cat(out, 1), both)
    f, a = rotary.frequencies(R, 10000.0)
    want = rotate(x, pos, f, a, layout)
    good &= bool(((both.cpu().double() - want).abs() <= half_step(want, dtype) + rotate_slack(x, layout, R, a)).all())
ok["rotary values"] = good
done("rotary")

for fmt, (B, first) in itertools.product(FORMATS, [(1, 0), (7, 3), (300, 5)]):
    old, new = [(i * 37) %% 60 for i in range(B)], [(i * 5 + 2) %% 7 for i in range(B)]
    size = 48 if fmt == "pools" else 16
    table, total = page_table([(a + n + size - 1) // size for a, n in zip(old, new)], 2, g)
    table[:, -1] = torch.where(torch.arange(B) %% 3 == 1, ints(-5).expand(B), table[:, -1])      # no page there
    kv = empty_cache(fmt, total, 2, 128, table, ints(*old), B, dev)
    T = first + sum(new) + 3
    qkv = canary((T, 7 * 128), torch.bfloat16)
    qkv.copy_(torch.randn(T, 7 * 128, generator=g))
    cu = (offsets(new) + first).to(dev)
    for layout, R in (("half", 128), ("half", 48), ("interleaved", 40)):
        rope = rotary.RotaryEmbedding(128, rotary_dim=R, layout=layout, device=dev)
        paged.append_tokens(qkv, kv, 3, rope, cu_new=cu, q_out=canary((T, 3, 128), torch.float16),
                            positions=torch.randint(0, 1 << 20, (T,), generator=g).to(dev))
    paged.append_tokens(qkv[:B], kv, 3, q_out=canary((B, 3, 128), torch.bfloat16))
    paged.read_tokens(kv, cu, T, starts=kv.seq_lens)
    for bad in [(5, 2, 9, 1), (-7, 100, -100, 3), (2 ** 31 - 1, -2 ** 31, 0, 9)]:
        wild = ints(*(bad * B)[:B + 1]).to(dev)
        paged.append_tokens(qkv, kv, 3, cu_new=wild, q_out=canary((T, 3, 128), torch.float16))
        paged.read_tokens(kv, wild, T)
    kv.seq_lens.copy_(torch.randint(-100, 200, (B,), generator=g, dtype=torch.int32))
    paged.append_tokens(qkv, kv, 3, cu_new=cu)
    done("tokens %%s %%d" %% (fmt, B))

for D, (B, longest, Hkv, G, most) in itertools.product((64, 128), [(1, 40001, 1, 4, 1), (1, 3000, 2, 32, 3), (150, 170, 2, 2, 4), (40, 3000, 3, 5, 2), (3, 900, 2, 4, 90)]):
    lens = torch.randint(0, longest + 1, (B,), generator=g).tolist()
    lens[0] = longest
    queries = [1] * B if most == 1 else torch.randint(0, most + 1, (B,), generator=g).tolist()
    table, total = page_table([(n + 15) // 16 for n in lens], 3, g)
    k, v = (quantise4(torch.randn(total, Hkv, 16, D, generator=g)) for _ in range(2))
    buf = canary((total, Hkv, 18, D), torch.uint8)
    buf.copy_(paged.pack_kv4(*k, *v))
    kv = paged.PagedKV4(buf, table.to(dev), ints(*lens).to(dev), B)
    T = sum(queries) + (0 if most == 1 else 5)
    q = canary((T, Hkv * G, D), torch.float16)
    q.copy_(torch.randn(T, Hkv * G, D, generator=g))
    cu = None if most == 1 else (offsets(queries) + 2).to(dev)
    out = kv.decode(q, D ** -0.5, cu_q=cu, out=canary(q.shape, torch.bfloat16))
    ok["finite %%d %%d %%d" %% (D, B, G)] = bool(torch.isfinite(out[0 if most == 1 else 2:T - (0 if most == 1 else 3)]).all())
    for bad in [(5, 2, 9, 1), (-7, 100, -100, 3), (2 ** 31 - 1, -2 ** 31, 0, 9)]:
        kv.decode(q, D ** -0.5, cu_q=ints(*(bad * B)[:B + 1]).to(dev), out=canary(q.shape, torch.float16))
    kv.page_table[:, ::2] = 1 << 20
    kv.seq_lens.copy_(torch.randint(-100, 2 * longest, (B,), generator=g, dtype=torch.int32))
    kv.decode(q, D ** -0.5, cu_q=cu, out=canary(q.shape, torch.float16), status=torch.zeros(1, dtype=torch.int32, device=dev))
    per = total // B
    if per:
        paged.PagedKV4(buf[:per * B], None, None, B).decode(q, D ** -0.5, cu_q=cu, out=canary(q.shape, torch.float16))
    done("attention %%d %%d %%d" %% (D, B, G))
print(json.dumps({"lib": str(_lib.LIB_PATH), "ok": ok, "violations": seen}))
'''


def test_no_index_leaves_its_range(cuda_device):
    from llm_inference_optimization_b200 import build
    env = dict(os.environ, SKV_B200_LIB=str(build.build(bounds=True)), PYTHONPATH=str(ROOT))
    proc = subprocess.run([sys.executable, "-c", DRIVER % {"root": str(ROOT)}], capture_output=True, text=True, timeout=900, cwd=ROOT, env=env)
    assert proc.returncode == 0, proc.stderr[-3000:]
    res = json.loads([l for l in proc.stdout.splitlines() if l.startswith("{")][-1])
    assert res["lib"].endswith("libskv_b200_bounds.so")
    assert res["violations"] == {} and all(res["ok"].values()), res
