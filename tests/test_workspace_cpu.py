"""The linears' scratch belongs to one call."""
import weakref

import torch

from diffuser_b200 import ops


def test_every_call_gets_scratch_of_its_own():
    cpu = torch.device("cpu")
    a, b = ops.workspace(cpu, 512), ops.workspace(cpu, 512)
    assert a.numel() == b.numel() == 512 and a.dtype == torch.uint8
    assert a.data_ptr() != b.data_ptr()
    # nothing keeps it behind the caller's back, nor hands it to a smaller call
    gone = weakref.ref(a)
    del a
    assert gone() is None
    assert ops.workspace(cpu, 64).numel() == 64 and ops.workspace(cpu, 0) is None
    ops.release_workspaces()
    assert (b.fill_(3) == 3).all()
