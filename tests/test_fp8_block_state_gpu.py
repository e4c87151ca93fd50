"""What the token block refuses leaves the state as it was."""

from __future__ import annotations

import pytest
import torch

from lesiondiffusion_mlx_b200 import fp8_block

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("shape,dtype,match", [((2, 3, 64), torch.float32, "float16 or bfloat16"),
                                               ((1, 3, 64), torch.float16, "activations must be")])
def test_a_refused_extension_writes_nothing(cuda_device, shape, dtype, match):
    block = fp8_block.Fp8TokenBlock(fp8_block.random_weights(64, 64, 2, 2, 32, 128), heads=2, kv_heads=2)
    state = block.new_state(2, 20, page=16)
    block.extend(torch.randn(2, 5, 64, device=cuda_device, dtype=torch.float16), state)
    before = [t.view(torch.uint8).clone() for t in state.cache], state.lengths.tolist(), state.written
    with pytest.raises(ValueError, match=match):
        block.extend(torch.randn(*shape, device=cuda_device, dtype=dtype), state)
    assert all(torch.equal(a, b.view(torch.uint8)) for a, b in zip(before[0], state.cache))
    assert (state.lengths.tolist(), state.written) == before[1:]
