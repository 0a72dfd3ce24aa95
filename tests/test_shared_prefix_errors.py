"""What the attention behind a shared prefix says when something is wrong that only the device can see."""
import ctypes

import pytest

from tokenizer_b200.kernels import ops


def test_an_unaligned_base_is_called_that(monkeypatch):
    """Reason 2 of a kernel whose blocks do not wait on one another."""
    value = ctypes.c_int(7 * 16 + 2)
    monkeypatch.setattr(ops, "_error_word", (value, 0))
    monkeypatch.setattr(ops, "_registered", {})
    with pytest.raises(ops.KernelError, match="shared_prefix_tcgen05: .*not aligned"):
        ops.raise_if_error()
    assert value.value == 0
