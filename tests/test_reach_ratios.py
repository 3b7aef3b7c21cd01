"""Calls of windowed and prefix attention with many q heads to a kv head pass the host's part, whichever
kernel takes them (CPU: in a process that sees no device, where a launch ends in an error)."""

from __future__ import annotations

import os
import pathlib
import subprocess
import sys

import pytest

PKG = pathlib.Path(__file__).resolve().parents[1] / "plastic-infer_amd"

CALLS = """
import sys
sys.path.insert(0, sys.argv[1])
import torch
from plastic_infer import _native as N
assert torch.cuda.device_count() == 0
name, heads = sys.argv[2], int(sys.argv[3])
lib, at, dim, rows = N.load(), 1 << 20, 128, 6
for dtype in (0, 1, 2):
    for cu in (None, at):
        print("dtype", dtype, "ragged", cu is not None, flush=True)
        shape = (rows if cu is None else 2, rows, heads, 1, dim, 16, 10, 1.0, dtype, at)
        if name == "prefix":
            need = N.query("pia_prefix_attention_workspace_bytes", rows, heads, dim)
            rc = lib.pia_prefix_attention(64 * at, at, heads * dim, at, at, at, 4, at, None, 1, at, 4, at,
                                          cu, None, *shape, need, None)
        else:
            need = N.query("pia_window_attention_workspace_bytes", dim)
            rc = lib.pia_window_attention(64 * at, at, heads * dim, at, at, at, 4, at, cu, None, 8, 0,
                                          *shape, need, None)
        assert rc > 0 and b"no ROCm-capable device" in lib.pia_last_error(), (rc, lib.pia_last_error())
print("done")
"""


@pytest.mark.parametrize("heads", [128, 129, 160, 256])
@pytest.mark.parametrize("name", ["prefix", "window"])
def test_ratio(name, heads):
    env = dict(os.environ, HIP_VISIBLE_DEVICES="-1", ROCR_VISIBLE_DEVICES="-1")
    run = subprocess.run([sys.executable, "-c", CALLS, str(PKG), name, str(heads)], env=env,
                         capture_output=True, text=True, timeout=120)
    assert run.returncode == 0 and run.stdout.endswith("done\n"), \
        (run.returncode, run.stdout[-60:], run.stderr[-300:])
