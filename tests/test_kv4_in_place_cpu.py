"""Outputs in place of their inputs have to have the same pitch: refused before any device is touched."""
import ctypes as C

import pytest
import torch

import x100b
from test_kv4_cpu import APPEND, ATTN, NORM, kv

P, OTHER = 1 << 20, 1 << 21   # aligned addresses that are never read


def append(**kw):
    return x100b.lib().x100q_kv4_append_dev(C.byref(kv()), C.byref(x100b.Kv4AppendArgs(**dict(APPEND, **kw))), None)


def attend(**kw):
    return x100b.lib().x100q_kv4_attn_dev(C.byref(kv()), C.byref(x100b.Kv4AttnArgs(**dict(ATTN, **kw))), None)


def norm(**kw):
    return x100b.lib().x100q_add_rmsnorm_q8_dev(C.byref(x100b.NormQ8Args(**dict(NORM, **kw))), None)


@pytest.mark.parametrize("call,other,same", [
    (append, dict(q=OTHER, q_out=OTHER, q_stride=1024, q_out_stride=512), dict(q=OTHER, q_out=OTHER, q_stride=1024, q_out_stride=1024)),
    (attend, dict(q=OTHER, out=OTHER, q_stride=512, out_stride=520), dict(q=OTHER, out=OTHER, q_stride=520, out_stride=520)),
    (norm, dict(x=OTHER, residual_out=OTHER, ldx=256, ldo=512), dict(x=OTHER, residual_out=OTHER, ldx=512, ldo=512)),
    (norm, dict(x=OTHER, ldr=512), dict(x=OTHER, ldr=512, ldo=512))])
def test_in_place_takes_one_pitch(call, other, same):
    assert call(**other) == x100b.X100_E_ARG
    if not torch.cuda.is_available():
        assert call(**same) == x100b.X100_E_NODEV             # past the checks, and no device here
