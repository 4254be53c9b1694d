"""Limits of drafted tokens and of scoring without a GPU: windows of layers that share a cache, nodes and sequences of a step, guesses that are too many, memory
that scoring holds."""
import contextlib
import random
import weakref
from types import SimpleNamespace

import pytest
import torch

from rocml_b200 import kernels
from rocml_b200.cache import SequenceCache
from rocml_b200.errors import KernelError, RocmlError


class _OnAnotherDevice(torch.Tensor):
    def get_device(self):
        return 5


def test_a_sink_on_another_device_is_refused():
    from test_tree import _attention
    with pytest.raises(KernelError, match="one device"):
        _attention(sink=torch.zeros(8).as_subclass(_OnAnotherDevice))
