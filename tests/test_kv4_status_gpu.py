"""What mlm_wait reports when a wait ran out and a position, length or count lies outside its cache:
the wait, whose outputs are lost."""
from __future__ import annotations

import ctypes
import os
import shutil
import subprocess

import numpy as np
import pytest

from metallm_b200 import TYPE_F16, TYPE_F32, MLMError
from tests.conftest import ROOT

pytestmark = pytest.mark.gpu

# the context's error word, as a kernel whose bounded wait ran out leaves it
SHIM = r'''
#include "mlm_internal.h"
extern "C" void record(mlm_ctx *c, int status) { *c->host_status = status; }
'''
TIMEOUT, SHAPE = -7, -2


@pytest.fixture(scope="module")
def record(tmp_path_factory):
    cuda = "/usr/local/cuda/include"
    if shutil.which("g++") is None or not os.path.isdir(cuda):
        pytest.skip("no host compiler or CUDA headers")
    d = tmp_path_factory.mktemp("record")
    (d / "shim.cpp").write_text(SHIM)
    so = str(d / "shim.so")
    subprocess.run(["g++", "-std=c++17", "-shared", "-fPIC", "-I", os.path.join(ROOT, "metallm_b200", "csrc"), "-I", cuda,
                    str(d / "shim.cpp"), "-o", so], check=True)
    shim = ctypes.CDLL(so)
    shim.record.argtypes = [ctypes.c_void_p, ctypes.c_int]
    return shim.record


@pytest.mark.parametrize("op", ["append", "read", "attend few", "attend many"])
@pytest.mark.parametrize("earlier", [TIMEOUT, 0])
def test_a_bad_position_does_not_hide_a_wait_that_ran_out(ctx, record, op, earlier):
    c = ctx.kv4_cache(1, 1, 32)
    buf = ctx.to_device(np.zeros(20 * 128 * 2, np.float32))
    out = [ctx.alloc(20 * 128 * 4) for _ in "kv"]
    for b in (c.k_buffer, c.v_buffer):
        ctx.call("mlm_memset", b, 0, b.nbytes)
    bad = ctx.to_device(np.array([33], np.int32))
    ctx.wait()
    record(ctx.handle, earlier)
    if op == "append":
        ctx.kv4_append(c, buf, buf, TYPE_F32, 128, 1, bad)
    elif op == "read":
        ctx.kv4_read_f16(c, 1, bad, None, *out)
    else:
        ctx.attn_kv4(c, buf, 1, 1 if op == "attend few" else 20, bad, None, out[0], TYPE_F16)
    with pytest.raises(MLMError) as e:
        ctx.wait()
    assert e.value.status == (earlier or SHAPE)
    ctx.wait()  # reported once
