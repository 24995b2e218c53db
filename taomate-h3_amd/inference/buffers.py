"""Buffers that belong to a kernel's input in the dtype they were made in."""

from __future__ import annotations

import torch.nn as nn


class FixedDtypeModule(nn.Module):
    """A module whose buffers named in ``FIXED`` go with it to another device, but keep their dtype where
    ``Module.to(dtype)``, ``half()`` or ``bfloat16()`` converts a model's floating tensors."""

    FIXED: tuple[str, ...] = ()

    def _apply(self, fn, recurse=True):
        held = {name: getattr(self, name) for name in self.FIXED}
        super()._apply(fn, recurse)
        for name, tensor in held.items():
            now = getattr(self, name)
            if tensor is not None and now.dtype != tensor.dtype:
                setattr(self, name, tensor.to(now.device))
        return self


__all__ = ["FixedDtypeModule"]
