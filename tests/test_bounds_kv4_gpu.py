"""The range-checking debug library runs rotation, append, read-back and 4-bit attention clean, outputs and caches between
canary bytes.  The library is chosen per process, so the driver runs in a child process; it prints one JSON line."""
import json
import os
import subprocess
import sys
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]
pytestmark = pytest.mark.gpu

DRIVER = r'''
import ctypes as C, json, sys
import torch
sys.path[:0] = [%(root)r, %(root)r + "/tests"]
from kv4_oracle import attend, half_step, ints, offsets, page_table, quantise4, values4
from llm_inference_optimization_b200 import _lib, paged, rotary
lib = _lib.load()
dev = torch.device("cuda", 0)
raws = []

def word(name):
    f = getattr(lib, name); f.restype = C.c_int; f.argtypes = [C.POINTER(C.c_int)]
    v = C.c_int(-1); assert f(C.byref(v)) == 0
    return v.value

def canary(shape, dtype):
    n = int(torch.tensor(shape).prod()) * torch.empty((), dtype=dtype).element_size()
    raw = torch.full((n + 8192,), 0xA5, dtype=torch.uint8, device=dev)
    raws.append(raw)
    return raw[4096:4096 + n].view(dtype).view(shape)

ok = {}
for D in (64, 128):
    g = torch.Generator().manual_seed(D)
    Hq, Hkv, lens, new = 6, 2, [300, 0, 77], [5, 40, 1]
    table, total = page_table([25, 25, 25], 2, g)
    buf = canary((total, Hkv, 18, D), torch.uint8)
    k, v = (quantise4(torch.randn(total, Hkv, 16, D, generator=g)) for _ in range(2))
    buf.copy_(paged.pack_kv4(*k, *v))
    kv = paged.PagedKV4(buf, table.to(dev), ints(*lens).to(dev), 3)
    T = sum(new)
    qkv = canary((T, (Hq + 2 * Hkv) * D), torch.float16)
    qkv.copy_(torch.randn(T, (Hq + 2 * Hkv) * D, generator=g))
    rope = rotary.RotaryEmbedding(D, rotary_dim=D // 2, device=dev)
    cu = offsets(new).to(dev)
    q = paged.append_tokens(qkv, kv, Hq, rope, cu_new=cu, q_out=canary((T, Hq, D), torch.float16))
    view = canary((T, Hq + Hkv, D), torch.float16)
    view.copy_(qkv.view(T, -1, D)[:, :Hq + Hkv])
    pos = torch.cat([torch.arange(a, a + n) for a, n in zip(lens, new)]).to(dev)
    rope.apply(pos, view[:, :Hq], view[:, Hq:], inplace=True)
    ok["rotary%%d" %% D] = torch.equal(view[:, :Hq], q)
    kv.seq_lens += ints(*new).to(dev)
    out = kv.decode(q, D ** -0.5, cu_q=cu, out=canary((T, Hq, D), torch.float16))
    kc, ks, vc, vs = (t.cpu() for t in paged.unpack_kv4(buf))
    good, at = True, 0
    for b, n in enumerate(new):
        t = torch.arange(lens[b] + n)
        row = lambda x: x.transpose(1, 2)[table[b, t // 16].long(), t %% 16]
        want, tol = attend(q[at:at + n].cpu(), values4(row(kc), row(ks)), values4(row(vc), row(vs)),
                           row(vs).double().repeat_interleave(32, -1), D ** -0.5, n)
        good &= bool(((out[at:at + n].cpu().double() - want).abs() <= tol + half_step(want, torch.float16)).all())
        at += n
    ok["attention%%d" %% D] = good
    K, V = paged.read_tokens(kv, cu, T, starts=ints(*lens).to(dev))
    ok["read%%d" %% D] = bool(torch.isfinite(K).all() and torch.isfinite(V).all())
torch.cuda.synchronize()
ok["canaries"] = all(bool((r[:4096] == 0xA5).all() and (r[-4096:] == 0xA5).all()) for r in raws)
print(json.dumps({"lib": str(_lib.LIB_PATH), "ok": ok,
                  "violations": {n: word("skv_debug_bounds_" + n) for n in ("kv_tokens", "gqa_decode_kv4")}}))
'''


def test_bounds_checked_library_runs_the_4_bit_path_without_a_violation(cuda_device):
    from llm_inference_optimization_b200 import build
    env = dict(os.environ, SKV_B200_LIB=str(build.build(bounds=True)), PYTHONPATH=str(ROOT))
    proc = subprocess.run([sys.executable, "-c", DRIVER % {"root": str(ROOT)}], capture_output=True, text=True, timeout=600, cwd=ROOT, env=env)
    assert proc.returncode == 0, proc.stderr[-3000:]
    res = json.loads([l for l in proc.stdout.splitlines() if l.startswith("{")][-1])
    assert res["lib"].endswith("libskv_b200_bounds.so")
    assert all(res["ok"].values()), res["ok"]
    assert all(v == 0 for v in res["violations"].values()), res["violations"]
