"""CPU tests of the 4-bit cache's and the sampler's argument checks: every refusal comes
before any CUDA call, so a context without a device sees them all."""
from __future__ import annotations

import ctypes
import os
import shutil
import subprocess

import numpy as np
import pytest

from tests import kv4_reference as R
from tests.conftest import ROOT

SHIM = r'''
#include "mlm_internal.h"
extern "C" mlm_ctx *bare_ctx() { mlm_ctx *c = new mlm_ctx(); c->sm_count = 148; return c; }
extern "C" void bare_free(mlm_ctx *c) { delete c; }
'''


@pytest.fixture(scope="module")
def bare(tmp_path_factory):
    """(library, context without a device or scratch)"""
    cuda = "/usr/local/cuda/include"
    if shutil.which("g++") is None or not os.path.isdir(cuda):
        pytest.skip("no host compiler or CUDA headers")
    d = tmp_path_factory.mktemp("bare")
    (d / "shim.cpp").write_text(SHIM)
    so = str(d / "shim.so")
    subprocess.run(["g++", "-std=c++17", "-shared", "-fPIC", "-I", os.path.join(ROOT, "metallm_b200", "csrc"), "-I", cuda,
                    str(d / "shim.cpp"), "-o", so], check=True)
    shim = ctypes.CDLL(so)
    shim.bare_ctx.restype = ctypes.c_void_p
    shim.bare_free.argtypes = [ctypes.c_void_p]
    from metallm_b200 import load
    lib = load()
    h = ctypes.c_void_p(shim.bare_ctx())
    yield lib, h
    shim.bare_free(h)


ARG, SHAPE, ALIGN, UNSUPPORTED = -1, -2, -3, -9
P = 0x10000  # an aligned address that no refused call may touch


def _cache(**kw):
    from metallm_b200 import Kv4Cache
    f = dict(k=P, v=2 * P, batch=2, n_kv_heads=4, head_dim=128, capacity=64)
    f.update(kw)
    return Kv4Cache(*(f[n] for n, _ in Kv4Cache._fields_))


BAD_CACHES = [(dict(k=None), ARG), (dict(v=None), ARG), (dict(head_dim=64), UNSUPPORTED), (dict(head_dim=0), UNSUPPORTED),
              (dict(batch=0), SHAPE), (dict(batch=-1), SHAPE), (dict(batch=1025), SHAPE), (dict(n_kv_heads=0), SHAPE),
              (dict(n_kv_heads=1025), SHAPE), (dict(capacity=0), SHAPE), (dict(capacity=(1 << 30) + 1), SHAPE),
              (dict(k=P + 8), ALIGN), (dict(v=P + 4), ALIGN)]


@pytest.mark.parametrize("bad,status", BAD_CACHES)
def test_every_call_refuses_a_bad_cache(bare, bad, status):
    lib, h = bare
    c = _cache(**bad)
    assert lib.mlm_kv4_append(h, c, P, P, 0, 512, 1, P, None) == status
    assert lib.mlm_kv4_read_f16(h, c, 1, P, None, P, P) == status
    assert lib.mlm_attn_kv4(h, c, P, 8, 1, P, None, P, 1) == status
    assert lib.mlm_last_error(h).decode().startswith("mlm_attn_kv4")


def test_null_context_and_cache(bare):
    lib, h = bare
    c = _cache()
    assert lib.mlm_kv4_append(None, c, P, P, 0, 512, 1, P, None) == ARG
    assert lib.mlm_kv4_read_f16(None, c, 1, P, None, P, P) == ARG
    assert lib.mlm_attn_kv4(None, c, P, 8, 1, P, None, P, 1) == ARG
    assert lib.mlm_sample_f32(None, P, 1, 8, 8, P, P, P, None) == ARG
    assert lib.mlm_kv4_append(h, None, P, P, 0, 512, 1, P, None) == ARG
    assert lib.mlm_attn_kv4(h, None, P, 8, 1, P, None, P, 1) == ARG


@pytest.mark.parametrize("args,status", [
    ((None, P, 0, 512, 1, P, None), ARG), ((P, None, 0, 512, 1, P, None), ARG), ((P, P, 0, 512, 1, None, None), ARG),
    ((P, P, 2, 512, 1, P, None), UNSUPPORTED), ((P, P, 12, 512, 1, P, None), UNSUPPORTED),
    ((P, P, 0, 511, 1, P, None), SHAPE), ((P, P, 0, -512, 1, P, None), SHAPE), ((P, P, 0, 1 << 40, 1, P, None), SHAPE),
    ((P, P, 0, 512, 0, P, None), SHAPE), ((P, P, 0, 512, 65, P, None), SHAPE), ((P, P, 0, 512, -1, P, None), SHAPE),
    ((P, P, 0, 514, 1, P, None), ALIGN), ((P, P, 1, 516, 1, P, None), ALIGN), ((P + 8, P, 0, 512, 1, P, None), ALIGN),
    ((P, P + 4, 30, 512, 1, P, None), ALIGN), ((P, P, 0, 512, 1, P + 2, None), ALIGN), ((P, P, 0, 512, 1, P, P + 1), ALIGN)])
def test_append_refusals(bare, args, status):
    lib, h = bare
    assert lib.mlm_kv4_append(h, _cache(), *args) == status


@pytest.mark.parametrize("args,status", [
    ((0, P, None, P, P), SHAPE), ((65, P, None, P, P), SHAPE), ((1, None, None, P, P), ARG), ((1, P, None, None, P), ARG),
    ((1, P, None, P, None), ARG), ((1, P, None, P + 8, P), ALIGN), ((1, P + 1, None, P, P), ALIGN)])
def test_read_refusals(bare, args, status):
    lib, h = bare
    assert lib.mlm_kv4_read_f16(h, _cache(), *args) == status


@pytest.mark.parametrize("args,status", [
    ((None, 8, 1, P, None, P, 1), ARG), ((P, 8, 1, None, None, P, 1), ARG), ((P, 8, 1, P, None, None, 1), ARG),
    ((P, 6, 1, P, None, P, 1), SHAPE), ((P, 0, 1, P, None, P, 1), SHAPE), ((P, -8, 1, P, None, P, 1), SHAPE),
    ((P, 1 << 20, 1, P, None, P, 1), SHAPE), ((P, 8, 0, P, None, P, 1), SHAPE), ((P, 8, 65537, P, None, P, 1), SHAPE),
    ((P, 8, 1, P, None, P, 0), UNSUPPORTED), ((P, 8, 1, P, None, P, 7), UNSUPPORTED), ((P + 2, 8, 1, P, None, P, 1), ALIGN),
    ((P, 8, 1, P, None, P + 2, 1), ALIGN), ((P, 8, 1, P + 2, None, P, 1), ALIGN), ((P, 8, 1, P, P + 2, P, 30), ALIGN)])
def test_attention_refusals(bare, args, status):
    lib, h = bare
    assert lib.mlm_attn_kv4(h, _cache(), *args) == status


@pytest.mark.parametrize("args,status", [
    ((None, 1, 8, 8, P, P, P, P), ARG), ((P, 1, 8, 8, None, P, P, P), ARG), ((P, 1, 8, 8, P, None, P, P), ARG),
    ((P, 1, 8, 8, P, P, None, P), ARG), ((P, 0, 8, 8, P, P, P, P), SHAPE), ((P, 65537, 8, 8, P, P, P, P), SHAPE),
    ((P, 1, 0, 8, P, P, P, P), SHAPE), ((P, 1, (1 << 22) + 1, 1 << 23, P, P, P, P), SHAPE), ((P, 2, 8, 7, P, P, P, P), SHAPE),
    ((P + 1, 1, 8, 8, P, P, P, P), ALIGN), ((P, 1, 8, 8, P, P, P + 2, P), ALIGN), ((P, 1, 8, 8, P, P, P, P + 2), ALIGN)])
def test_sample_refusals(bare, args, status):
    lib, h = bare
    assert lib.mlm_sample_f32(h, *args) == status


def test_quantizer_holds_values_within_half_a_step():
    """The format itself: |value - x| is at most half a step plus the fp16 roundings of m and d."""
    rng = np.random.default_rng(0)
    x = rng.standard_normal((50, R.D)).astype(np.float32) * 10.0 ** rng.integers(-3, 4, (50, 1))
    v = R.values(R.quantize(x.astype(np.float32)))
    g = x.reshape(50, 4, 32)
    span = (g.max(-1) - g.min(-1))[..., None]
    # m is off by 2^-11 of the minimum, d by 2^-11 of itself times up to 15 steps
    bound = span / 30 + 2.0 ** -10 * (np.abs(g.min(-1))[..., None] + span) + 2.0 ** -20
    assert np.all(np.abs(v.reshape(50, 4, 32) - g) <= bound)


def test_params_array_is_the_struct():
    from metallm_b200 import SampleParams, sample_params
    a = sample_params([(0.5, 40, 0.9, 0.1), (0.0, 0, 1.0, 0.0)])
    assert a.itemsize == ctypes.sizeof(SampleParams) == 16
    s = SampleParams.from_buffer_copy(a[:1].tobytes())
    assert (s.temperature, s.top_k) == (0.5, 40) and abs(s.top_p - 0.9) < 1e-7
