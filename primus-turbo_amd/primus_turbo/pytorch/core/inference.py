"""What the inference operators check of their tensors, apart from shapes and types."""

from __future__ import annotations

from typing import Optional, Sequence

import torch
from torch._subclasses.fake_tensor import FakeTensor
from torch.autograd import forward_ad

__all__ = ["check_tensors", "refuse_gradients"]


def refuse_gradients(what: str, *tensors: Optional[torch.Tensor]) -> None:
    """What asks for a derivative of an inference operator gets an error, not a
    result without one."""
    if torch.is_grad_enabled():
        assert not any(t is not None and t.requires_grad for t in tensors), (
            f"{what} has no backward pass: call it under torch.no_grad() or on detached tensors"
        )
    if forward_ad._current_level >= 0:
        for t in tensors:
            if t is not None:
                assert forward_ad.unpack_dual(t).tangent is None, f"{what} has no forward-mode derivative"


def check_tensors(what: str, floats: Sequence[Optional[torch.Tensor]], *others: torch.Tensor) -> None:
    """No derivative is asked for with respect to ``floats`` (what the result depends
    on); all tensors are on one device, and that a GPU: kernels get raw pointers.
    These calls are made token by token: one look at each tensor where all is well."""
    dev = floats[0].get_device()
    # one is enough: they do not go together with tensors that have memory
    assert not isinstance(floats[0], FakeTensor), f"{what} runs on memory: fake tensors have none"
    if dev >= 0 and forward_ad._current_level < 0:
        for t in floats:
            if t is not None and (t.requires_grad or t.get_device() != dev):
                break
        else:
            for t in others:
                if t.get_device() != dev:
                    break
            else:
                return
    refuse_gradients(what, *floats)
    first = floats[0].device
    assert all(t is None or t.device == first for t in (*floats, *others)), f"all tensors must be on {first}"
    # without a GPU the launch says that there is none
    assert dev >= 0 or not torch.cuda.is_available(), f"all tensors must be GPU tensors, got {first}"
