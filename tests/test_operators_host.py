"""What the operators' Python side does on the host: no GPU, the device's words are set by hand."""

import pytest
import torch

from cohere_inference_b200 import native as nv
from cohere_inference_b200.packing import W8A8Linear


def test_w8a8_status_is_reported_once():
    lin = object.__new__(W8A8Linear)
    lin.status = torch.zeros(1, dtype=torch.int32)
    lin.check_status()
    lin.status |= nv.ST_TIMEOUT
    with pytest.raises(nv.NativeError, match="ran out"):
        lin.check_status()
    assert int(lin.status) == 0
    lin.check_status()
