"""Results of the performance cases' passes are the caller's: they outlive the state that a pass ran on."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

CODE = """
import gc, weakref
import torch
from perf import operators as ops
ops.own = True
cases = [dict(kind="embed_grad", M=700, V=300, H=64, dy="bf16", dense=False, pad=0.0, skip=0.05, scale=1.0),
         dict(kind="dispatch", T=300, k=2, E=5, H=64, type="bf16", align=16, mask=0.1, back=False)]
for c in cases:
    state = ops.prepare(c, 1)
    got = ops.run(state)
    torch.cuda.synchronize()
    want, owner, kept = {n: t.clone() for n, t in got.items()}, state.kept.owner, weakref.ref(state.kept)
    del state
    gc.collect()
    assert owner._block is not None, "freed under its tensors"
    for seed in (2, 3):                                # other states come and go
        ops.run(ops.prepare(c, seed))
    torch.cuda.synchronize()
    for n, t in got.items():
        assert torch.equal(t, want[n]), (c["kind"], n)
    del got, t
    gc.collect()
    assert kept() is None and owner._block is None, "never freed"
    print(c["kind"], "ok", flush=True)
"""


def test_results_outlive_their_state():
    pytest.importorskip("torch")
    r = subprocess.run([sys.executable, "-c", CODE], cwd=ROOT, capture_output=True, text=True, timeout=110)
    assert r.returncode == 0 and r.stdout.split("\n")[:2] == ["embed_grad ok", "dispatch ok"], r.stdout + r.stderr
