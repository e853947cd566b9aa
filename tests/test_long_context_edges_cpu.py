"""GPU-less checks of what attention over long contexts takes and refuses, where the usual cases do not go."""
import pytest

from test_long_context_cpu import _calls, here  # noqa: F401
from test_attention_cpu import _cache


@pytest.mark.parametrize("axes", [1, 2, 4])
def test_axes_may_share_their_positions(axes):
    """A stride of 0 is no error (what is, of the other arguments, still comes up): positions are only read."""
    import pplb200
    c = _calls()
    for stride in (0, 4, 5):
        assert c["rotary"](dict(axes=axes, stride=stride), tokens=0) == c["write"](_cache(), dict(axes=axes, stride=stride), tokens=0) == 0
        assert c["write"](_cache(), dict(axes=axes, stride=stride), rd=0) == 4
        assert "overlap" not in pplb200.last_error()
    if axes > 1:
        assert c["write"](_cache(), dict(axes=axes, stride=3), rd=0) == 4 and "overlap" in pplb200.last_error()


def test_binding_takes_expanded_positions(here):  # noqa: F811
    import struct

    import torch
    import pplb200
    table = pplb200.RotaryTable(64, device="cpu", axes=(16, 8, 8))
    for tokens in (1, 5):
        pos = torch.zeros(tokens, dtype=torch.int64).expand(3, -1)
        pplb200.rotary_fp16(torch.zeros((tokens, 4, 64), dtype=torch.float16), None, pos, table)
        assert struct.unpack("=Qq2i", here[-1][1][-1]) == (table.axis_of_plane.data_ptr(), 0, 3, 0)
