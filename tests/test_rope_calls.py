"""swq_rope_table and swq_rope without a GPU: what they refuse before they touch a device, and a config's settings."""

import ctypes
import math

import pytest

from swiftlet_amd import _lib
from swiftlet_amd._lib import RopeHeads, RopeScalingDesc
from swiftlet_amd.rope import RopeGPU, RopeScaling

FAKE = 0x7F0000000000  # a well-aligned address; a refused call uses none
E = _lib


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def scaling(**kw):
    d = dict(kind=E.SWQ_ROPE_YARN, original_positions=4096, beta_fast=32.0, beta_slow=1.0, magnitude=0.0, factor=4.0, reserved=0)
    return RopeScalingDesc(**{**d, **kw})


def table(lib, sc=None, rot=64, theta=1e7, positions=None, first=0, count=5, out=FAKE):
    return lib.swq_rope_table(rot, theta, ctypes.byref(sc) if sc else None, positions, first, count, out, None)


@pytest.mark.parametrize("kw,want", [
    (dict(rot=0), E.SWQ_ERR_BAD_SHAPE), (dict(rot=7), E.SWQ_ERR_BAD_SHAPE), (dict(rot=514), E.SWQ_ERR_LIMIT), (dict(theta=0.0), E.SWQ_ERR_INVALID_ARGUMENT),
    (dict(theta=math.inf), E.SWQ_ERR_INVALID_ARGUMENT), (dict(theta=math.nan), E.SWQ_ERR_INVALID_ARGUMENT), (dict(count=-1), E.SWQ_ERR_INVALID_ARGUMENT),
    (dict(out=None), E.SWQ_ERR_INVALID_ARGUMENT), (dict(out=FAKE + 4), E.SWQ_ERR_MISALIGNED), (dict(positions=FAKE + 2), E.SWQ_ERR_MISALIGNED)], ids=str)
def test_table(lib, kw, want):
    assert table(lib, **kw) == want


@pytest.mark.parametrize("kw,rot,want", [
    (dict(kind=4), 64, E.SWQ_ERR_INVALID_ARGUMENT), (dict(kind=-1), 64, E.SWQ_ERR_INVALID_ARGUMENT), (dict(factor=0.0), 64, E.SWQ_ERR_INVALID_ARGUMENT),
    (dict(factor=math.nan), 64, E.SWQ_ERR_INVALID_ARGUMENT), (dict(factor=-2.0, kind=E.SWQ_ROPE_LINEAR), 64, E.SWQ_ERR_INVALID_ARGUMENT),
    (dict(kind=E.SWQ_ROPE_NTK), 2, E.SWQ_ERR_BAD_SHAPE), (dict(original_positions=0), 64, E.SWQ_ERR_INVALID_ARGUMENT), (dict(beta_fast=0.0), 64, E.SWQ_ERR_INVALID_ARGUMENT),
    (dict(beta_slow=-1.0), 64, E.SWQ_ERR_INVALID_ARGUMENT), (dict(beta_fast=math.inf), 64, E.SWQ_ERR_INVALID_ARGUMENT),
    (dict(magnitude=-1.0), 64, E.SWQ_ERR_INVALID_ARGUMENT), (dict(magnitude=math.inf), 64, E.SWQ_ERR_INVALID_ARGUMENT), (dict(reserved=1), 64, E.SWQ_ERR_INVALID_ARGUMENT)], ids=str)
def test_scalings(lib, kw, rot, want):
    assert table(lib, scaling(**kw), rot=rot) == want


def test_no_rows_need_nothing(lib):
    assert table(lib, count=0, out=None) == E.SWQ_OK
    assert table(lib, scaling(), count=0, out=None) == E.SWQ_OK


def heads(**kw):
    d = dict(x=FAKE, out=FAKE + (1 << 32), token_stride=4096, head_stride=256, out_token_stride=4096, out_head_stride=256, norm_weight=FAKE, heads=16, reserved=0)
    return RopeHeads(**{**d, **kw})


def turn(lib, *parts, n=None, tokens=9, hd=256, rot=64, layout=0, inverse=0, eps=1e-6, t=FAKE, rows_of=9, rows=None, dtype=E.SWQ_BF16):
    arr = (RopeHeads * max(len(parts), 1))(*parts)
    return lib.swq_rope(arr, len(parts) if n is None else n, tokens, hd, rot, layout, inverse, eps, t, rows_of, rows, dtype, None)


@pytest.mark.parametrize("kw,want", [
    (dict(n=0), E.SWQ_ERR_INVALID_ARGUMENT), (dict(n=-1), E.SWQ_ERR_INVALID_ARGUMENT), (dict(n=5), E.SWQ_ERR_LIMIT), (dict(tokens=-1), E.SWQ_ERR_INVALID_ARGUMENT),
    (dict(hd=0), E.SWQ_ERR_BAD_SHAPE), (dict(hd=513), E.SWQ_ERR_LIMIT), (dict(rot=0), E.SWQ_ERR_BAD_SHAPE), (dict(rot=63), E.SWQ_ERR_BAD_SHAPE),
    (dict(rot=258), E.SWQ_ERR_BAD_SHAPE), (dict(layout=2), E.SWQ_ERR_INVALID_ARGUMENT), (dict(inverse=2), E.SWQ_ERR_INVALID_ARGUMENT),
    (dict(eps=math.nan), E.SWQ_ERR_INVALID_ARGUMENT), (dict(dtype=E.SWQ_F16), E.SWQ_ERR_UNSUPPORTED_DTYPE), (dict(t=None), E.SWQ_ERR_INVALID_ARGUMENT),
    (dict(t=FAKE + 4), E.SWQ_ERR_MISALIGNED), (dict(rows_of=0), E.SWQ_ERR_INVALID_ARGUMENT), (dict(rows_of=8), E.SWQ_ERR_BAD_SHAPE),
    (dict(rows=FAKE + 2), E.SWQ_ERR_MISALIGNED), (dict(tokens=1 << 23, rows=FAKE), E.SWQ_ERR_LIMIT)], ids=str)
def test_turns(lib, kw, want):
    assert turn(lib, heads(), **kw) == want


@pytest.mark.parametrize("kw,want", [
    (dict(x=None), E.SWQ_ERR_INVALID_ARGUMENT), (dict(out=None), E.SWQ_ERR_INVALID_ARGUMENT), (dict(x=FAKE + 1), E.SWQ_ERR_MISALIGNED),
    (dict(out=FAKE + 3), E.SWQ_ERR_MISALIGNED), (dict(norm_weight=FAKE + 2), E.SWQ_ERR_MISALIGNED), (dict(heads=0), E.SWQ_ERR_INVALID_ARGUMENT),
    (dict(reserved=1), E.SWQ_ERR_INVALID_ARGUMENT), (dict(heads=65537), E.SWQ_ERR_LIMIT)], ids=str)
def test_heads(lib, kw, want):
    assert turn(lib, heads(), heads(**kw)) == want


def test_no_tokens_need_nothing(lib):
    assert turn(lib, heads(x=None, out=None), tokens=0, t=None, rows_of=0) == E.SWQ_OK


def test_config():
    base = dict(head_dim=256, partial_rotary_factor=0.25, rope_theta=1e6, max_position_embeddings=4096)
    r = RopeGPU.from_config(base, device="cpu")
    assert (r.rot, r.theta, r.scaling) == (64, 1e6, None)
    r = RopeGPU.from_config({**base, "rope_scaling": {"type": "yarn", "factor": 4.0}}, device="cpu")
    assert r.scaling == RopeScaling("yarn", 4.0, 4096)
    r = RopeGPU.from_config({"text_config": dict(head_dim=128, rope_parameters=dict(
        rope_type="yarn", rope_theta=5e6, partial_rotary_factor=0.5, factor=2.0, original_max_position_embeddings=8192, beta_fast=16, attention_factor=1.5))}, device="cpu")
    assert (r.rot, r.theta, r.scaling) == (64, 5e6, RopeScaling("yarn", 2.0, 8192, 16.0, 1.0, 1.5))
    with pytest.raises(_lib.SwqError):
        RopeGPU.from_config({**base, "rope_scaling": {"rope_type": "something"}}, device="cpu")
    yarn = {"rope_type": "yarn", "factor": 4.0}
    for odd in ({"mscale": 1.0}, {"mscale_all_dim": 0.7}, {"truncate": False}):
        with pytest.raises(_lib.SwqError):
            RopeGPU.from_config({**base, "rope_scaling": {**yarn, **odd}}, device="cpu")
    assert RopeGPU.from_config({**base, "rope_scaling": {**yarn, "truncate": True, "mscale": None}}, device="cpu").scaling == RopeScaling("yarn", 4.0, 4096)
    with pytest.raises(_lib.SwqError):
        RopeGPU(64, 1e6, layout="other")
    with pytest.raises(_lib.SwqError):
        RopeGPU(64, 1e6, scaling=RopeScaling("other", 2.0))
