"""Handles of 4-bit weights and the life of their context."""
import numpy as np
import pytest

from test_q4_gpu import weights

pytestmark = pytest.mark.gpu


def test_a_weight_may_outlive_its_context():
    """Destroying the context first leaves a handle that can only be destroyed; its memory comes back."""
    import torch
    import shainet_b200 as S
    from shainet_b200 import build
    build.build()
    c = S.AttnContext(0)
    rng = np.random.default_rng(1)
    packed, scales = weights(rng, 4096, 32768, 32)
    before = torch.cuda.mem_get_info()[0]
    W = S.Q4Weight.from_quantized(c, packed, scales, 4096, 32)
    held = torch.cuda.mem_get_info()[0]
    assert before - held >= 64 << 20
    c.close()
    W.close()
    assert torch.cuda.mem_get_info()[0] - held >= 64 << 20
