"""Checks that the inference operators share.  They are called token by token, so
each is kept to what it costs."""

from __future__ import annotations

from typing import Optional

import torch

__all__ = ["check_devices"]


def check_devices(*tensors: Optional[torch.Tensor]) -> None:
    """All on the first one's device, and that a GPU's: kernels get raw pointers."""
    dev = tensors[0].get_device()
    for t in tensors:
        if t is not None and (t.get_device() != dev or dev < 0):
            first = tensors[0].device
            assert all(x is None or x.device == first for x in tensors), f"all tensors must be on {first}"
            # without a GPU the launch says that there is none
            assert not torch.cuda.is_available(), f"all tensors must be GPU tensors, got {first}"
            return
