"""The binding of a block's adapters, without a device."""
import pytest

import qimm


def test_a_projection_that_no_block_has_is_refused():
    """ctypes would take the name as an attribute of its own and the adapter would be lost."""
    blk = object.__new__(qimm.Block)  # refused before the library is called
    pair = (qimm.BF16, 128, 64, 1, bytes(128), bytes(256))
    for name in ("down", "gate", "to_out.0"):
        with pytest.raises(qimm.QimmError, match=name):
            blk.set_adapters([(1.0, {"to_q": pair, name: pair})])
