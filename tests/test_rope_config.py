"""Scalings of a config.json that leaves settings out or has null for them."""

import pytest

from swiftlet_amd import _lib
from swiftlet_amd.rope import RopeGPU, RopeScaling

BASE = dict(head_dim=256, partial_rotary_factor=0.25, rope_theta=1e6, max_position_embeddings=4096)


@pytest.mark.parametrize("kind", ["linear", "ntk", "yarn"])
@pytest.mark.parametrize("factor", [{}, {"factor": None}], ids=["none", "null"])
def test_no_factor(kind, factor):
    for key in ("rope_scaling", "rope_parameters"):
        with pytest.raises(_lib.SwqError) as e:
            RopeGPU.from_config({**BASE, key: {"rope_type": kind, **factor}}, device="cpu")
        assert e.value.code == _lib.SWQ_ERR_INVALID_ARGUMENT


def test_null_is_the_default():
    sc = dict(rope_type="yarn", factor=4.0, beta_fast=None, beta_slow=None, original_max_position_embeddings=None, attention_factor=None, mscale=None,
              mscale_all_dim=None, truncate=None)
    assert RopeGPU.from_config({**BASE, "rope_scaling": sc}, device="cpu").scaling == RopeScaling("yarn", 4.0, 4096)


def test_plain_needs_no_factor():
    assert RopeGPU.from_config({**BASE, "rope_scaling": {"rope_type": "default"}}, device="cpu").scaling is None
