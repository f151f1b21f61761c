"""Arguments of the quantiser's form for products, and of the layers (no kernel is launched in this file)."""
import ctypes
import os
import re

import pytest
import torch

from mor_b200 import cabi

HEADER = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "mor_b200.h")


def test_operand_formats_are_checked_like_the_others():
    assert re.search(r"#define MOR_B200_MX_OPERAND %d\b" % cabi.MX_OPERAND, open(HEADER).read())
    q, buf = cabi.lib().mor_b200_quantize_mx, ctypes.create_string_buffer(4096)
    p = (ctypes.addressof(buf) + 15) & ~15
    for fmt in (2, 4, -1, 15, 17 + 1, 16 + 4, 16 + 16, 1 << 20):        # E3M2 and E2M1 are no byte formats
        assert q(p, p, p, 4, 64, 32, fmt, None) == -1, fmt
    for fmt in (0, 1, 3):
        assert q(p, p, p, 4, 64, 48, 16 + fmt, None) == -1
        assert q(p + 2, p, p, 4, 64, 32, 16 + fmt, None) == -2 and q(p, p + 4, p, 4, 64, 32, 16 + fmt, None) == -2
        assert q(None, p, p, 4, 64, 32, 16 + fmt, None) == -1 and q(p, p, p, 0, 64, 32, 16 + fmt, None) == -1


@pytest.mark.parametrize("name,types", [("e4m3", (torch.bfloat16,)), ("e5m2", (torch.bfloat16,)), ("e2m1", (torch.bfloat16, torch.float32))])
def test_a_layer_is_made_of_types_that_its_quantiser_takes(name, types):
    """refused when it is made, not at its first call"""
    from mor_b200.nn import MXLinear
    for dtype in (torch.bfloat16, torch.float32, torch.float16, torch.float64, None):
        if (dtype or torch.get_default_dtype()) in types:
            assert MXLinear(64, 32, dtype=dtype, elem_format=name).weight.dtype == (dtype or torch.get_default_dtype())
        else:
            with pytest.raises(ValueError, match="dtype"):
                MXLinear(64, 32, dtype=dtype, elem_format=name)
