"""New outputs and workspaces are allocations that torch's dispatch modes see (no GPU: the mode stops the call there)."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.utils._python_dispatch import TorchDispatchMode

from dscuda_b200 import flash, mla


class Seen(Exception):
    pass


class Watch(TorchDispatchMode):
    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        if func is torch.ops.aten.empty.memory_format:
            raise Seen(f"{list(args[0])} {kwargs['device']}")
        return func(*args, **(kwargs or {}))


def fake(*shape, dtype=torch.bfloat16):
    with FakeTensorMode():
        return torch.empty(shape, dtype=dtype, device="cuda:0")


CALLS = {
    "mla_forward": lambda: (mla.mla_forward, fake(1, 3, 2, 512), fake(1, 3, 2, 64), fake(1, 3, 512), fake(1, 3, 64), 0.1),
    "prefill_forward": lambda: (mla.prefill_forward, fake(1, 5, 2, 128), fake(1, 5, 2, 64), fake(1, 5, 2, 128), fake(1, 5, 1, 64), fake(1, 5, 2, 128), 0.1),
    "absorb_query": lambda: (mla.absorb_query, fake(4, 2, 128), fake(256, 512)),
    "flash_forward": lambda: (mla.flash_forward, fake(1, 64, 4, 128), fake(1, 64, 2, 128), fake(1, 64, 2, 128), 0.1),
    "rope": lambda: (flash.rope, fake(4, 2, 128), None, fake(1, 4, dtype=torch.int32), [64]),
    "cross_forward": lambda: (flash.cross_forward, fake(1, 50, 4, 128), fake(1, 60, 2, 128), fake(1, 60, 2, 128), 0.1),
}


@pytest.mark.parametrize("name", CALLS)
def test_dispatch_modes_see_new_tensors(name):
    call, *arguments = CALLS[name]()
    with pytest.raises(Seen, match="cuda"), Watch():
        call(*arguments)
