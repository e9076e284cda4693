"""The measured operators' own calls against their plain forms, at sizes of a test: shapes, types and values."""
import importlib.util
import os
import sys

import pytest
import torch

pytestmark = pytest.mark.gpu

_REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture()
def cases():
    spec = importlib.util.spec_from_file_location("more_operators", os.path.join(_REPO, "perf", "more_operators.py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    yield module
    sys.modules.pop("more_operators", None)


def both(cases, case, seed=3):
    """(the plain form's outputs, the library's) on the same inputs."""
    outs = []
    for own in (False, True):
        cases.own = own
        outs.append(cases.run(cases.prepare(case, seed)))
    return outs


@pytest.mark.parametrize("dtype,master", [("bf16", False), ("bf16", True), ("f16", False), ("f32", False)])
@pytest.mark.parametrize("bits", [8, 32])
def test_adamw(dev, cases, dtype, master, bits):
    plain, own = both(cases, cases._adamw(None, 2, 45, 33, dtype, bits, master=master, clip=True))
    assert plain.keys() == own.keys()
    assert (plain["masters"] is None) == (own["masters"] is None) == (not master or dtype == "f32")
    for a, b in zip(plain["moments"], own["moments"]):
        # the same operations in the same order of fp32, the same numbers for the rounding
        assert a.shape == b.shape and a.dtype == b.dtype and torch.equal(a, b)
    for a, b in zip(plain["masters"] or plain["params"], own["masters"] or own["params"]):
        assert a.shape == b.shape and a.dtype == b.dtype
        # either is off by 12 roundings of the change (under 0.1) and 3 of the value, and half a step of its type
        size = a.float().abs() + 0.1
        assert bool(((a.float() - b.float()).abs() <= 2 * 15 * 2.0**-24 * size + torch.finfo(a.dtype).eps * size).all())
