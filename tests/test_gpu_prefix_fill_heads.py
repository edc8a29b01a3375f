"""A prefix fill into a cache of other heads than the blocks' is refused before any launch: their
keys and values would not fit it."""
import numpy as np
import pytest

import oracle as O
import qimm
from gpu_util import dev, host, stream
from test_gpu_block import SMALL
from test_gpu_step import JD, Built, model_weights

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["kv_create", "kv_create_host", "kv_create_q4"])
def test_other_heads_are_refused(torch_cuda, qctx, kind):
    torch, text, layers = torch_cuda, 24, 2
    mdl = Built(qctx, *model_weights(51, layers))
    txt = dev(torch, np.random.default_rng(1).standard_normal((1, text, JD)).astype(np.float32))
    pe, ids = dev(torch, O.rope_table([], [0] * text)), dev(torch, np.full(text, -1, np.int32))

    def fill(heads):
        kv = getattr(qctx, kind)(layers, 1, heads, text)
        try:
            mdl.model.prefix_fill(txt.data_ptr(), text, None, 0, 1, qimm.joint_layout_pieces(text), ids.data_ptr(), None,
                                  pe.data_ptr(), kv, stream(torch))
            k, v = (torch.empty(1, heads, text, 128, dtype=torch.bfloat16, device="cuda") for _ in range(2))
            kv.load(layers - 1, k.data_ptr(), v.data_ptr(), stream(torch))
            return host(k.float())
        finally:
            torch.cuda.synchronize()
            kv.free()

    for heads in (SMALL["heads"] - 1, SMALL["heads"] + 1):
        with pytest.raises(qimm.QimmError, match="QIMM_ERR_SHAPE"):
            fill(heads)
    assert np.isfinite(fill(SMALL["heads"])).all()
    mdl.free()
