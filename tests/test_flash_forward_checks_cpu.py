"""What the causal grouped-query forward refuses before anything is launched, on tensors without storage."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from dscuda_b200 import flash

MISSING = "[Dd]river|data pointer|storage|[Nn]o CUDA|NVIDIA"


def fake(*shape, dtype=torch.bfloat16, device="cuda:0"):
    with FakeTensorMode():
        return torch.empty(shape, dtype=dtype, device=device)


def call(query=(2, 70, 8, 128), key=(2, 70, 2, 128), value=(2, 70, 2, 128), **given):
    return flash.forward(*[fake(*shape, **given.get(name, {})) for name, shape in (("query_", query), ("key_", key), ("value_", value))], 0.1)


@pytest.mark.parametrize("given,message", [
    (dict(key=(2, 69, 2, 128)), "the key has fewer"), (dict(value=(2, 40, 2, 128)), "the value has fewer"), (dict(value=(2, 70, 1, 128)), "the value has fewer"),
    (dict(key=(1, 70, 2, 128)), "the key has fewer"), (dict(key=(2, 70, 2, 64)), "the key has fewer"),
    (dict(query_=dict(dtype=torch.float16)), "the query has the wrong dtype"), (dict(key_=dict(dtype=torch.float32)), "the key has the wrong dtype"),
    (dict(value_=dict(device="cuda:1")), "the value is on another device"), (dict(key=(140, 2, 128)), "4 dimensions"),
])
def test_refused(given, message):
    with pytest.raises(ValueError, match=message):
        call(**given)


@pytest.mark.parametrize("given", [{}, dict(query=(1, 70, 8, 128), key=(1, 90, 2, 128), value=(1, 90, 2, 128)), dict(value=(2, 70, 256))])
def test_accepted(given):
    with pytest.raises(RuntimeError, match=MISSING):
        call(**given)
