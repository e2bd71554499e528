"""Norm and rotation of heads (chk_qk_norm_rope) where a row's size and the weights' are far apart."""

from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

from cherenkov_amd import abi
from cherenkov_amd.abi import check, lib
from tests import step_ref as ref
from tests.test_gpu_kv4 import KINDS, dev, rounded, torch_type
from tests.test_gpu_step import turns

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("hd,rot", [(64, 64), (128, 32), (256, 20)])
@pytest.mark.parametrize("size,weight", [(2.0**50, 2.0**100), (2.0**-45, 2.0**-100), (2.0**50, 2.0**-60), (2.0**-45, 2.0**90)])
def test_weights_far_from_a_rows_size(have_gpu, kind, hd, rot, size, weight):
    """A dim times its weight is not f32's (2^150, 2^-145), the normed dim times it is."""
    import torch

    rng = np.random.default_rng(hd)
    nh, nkv, rows, eps = 3, 2, 70, 2.0**-100
    x, t = rounded(rng.normal(0, size, (rows, (nh + nkv) * hd)), kind)
    w, wt = rounded(rng.normal(1, 0.3, (2, hd)) * weight, "bf16")
    pos, tt = rng.integers(0, 9999, rows).astype(np.uint32), turns(1e4, rot)
    pos_t = dev(pos)
    norm = abi.ChkQkNorm(wt[0].data_ptr(), wt[1].data_ptr(), tt.data_ptr(), rot, nh, nkv, hd, 0, eps)
    out = torch.zeros(rows, (nh + nkv) * hd, dtype=torch_type(kind), device="cuda")
    check(lib().chk_qk_norm_rope(C.byref(norm), pos_t.data_ptr(), rows, t.data_ptr(), t.stride(0), out.data_ptr(), out.stride(0),
                                 t[:, nh * hd:].data_ptr(), t.stride(0), out[:, nh * hd:].data_ptr(), out.stride(0), KINDS[kind],
                                 None))
    torch.cuda.synchronize()
    got = out.double().cpu().numpy().reshape(rows, nh + nkv, hd)
    for heads, weights in ((slice(0, nh), w[0]), (slice(nh, nh + nkv), w[1])):
        want, big = ref.norm_rope(x.reshape(rows, nh + nkv, hd)[:, heads], weights, eps, pos, 1e4, rot)
        assert np.all(np.abs(got[:, heads] - want) <= ref.norm_rope_tolerance(kind, want, big))
