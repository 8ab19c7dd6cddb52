"""Which tensors a derived weight was made from: the layers keep concatenated or quantised copies of their projections'
weights and make them again when a source changes.

No counterpart in the reference, whose layers multiply with the projections as they are.
"""
from __future__ import annotations

import weakref
from typing import Optional, Sequence

import torch
from torch.multiprocessing.reductions import StorageWeakRef


class WeightSources:
    """The tensors behind a derived weight, without keeping them alive.

    ``same(tensors)`` is true while each is the very same tensor object over the very same storage, at the same
    place in it and written by no counted in-place operation since.  Objects and storages are held by weak references,
    so another tensor at a freed one's address, or other values moved to a freed storage's address, are told
    apart (addresses and version numbers alone repeat).  Writes that bypass the version counter (``t.data.copy_``) are
    not seen: call the layer's ``refresh_weights()`` after them."""

    def __init__(self, tensors: Sequence[Optional[torch.Tensor]] = ()) -> None:
        self._held = [None if t is None else (weakref.ref(t), StorageWeakRef(t.untyped_storage()), self._state(t))
                      for t in tensors]

    @staticmethod
    def _state(t: torch.Tensor):
        return t._version, t.dtype, t.storage_offset(), t.shape, t.stride()

    def same(self, tensors: Sequence[Optional[torch.Tensor]]) -> bool:
        if len(tensors) != len(self._held):
            return False
        for t, h in zip(tensors, self._held):
            if t is None or h is None:
                if t is not h:
                    return False
            elif h[0]() is not t or h[1].cdata != t.untyped_storage()._cdata or h[2] != self._state(t):
                return False
        return True

    # a copied or loaded layer has tensors of its own: its derived weights are made again
    def __deepcopy__(self, memo) -> "WeightSources":
        return WeightSources()

    def __copy__(self) -> "WeightSources":
        return WeightSources()

    def __reduce__(self):
        return WeightSources, ()
