"""Arguments of AdamW that its kernels cannot take, refused before a tensor is touched (no GPU needed)."""

import pytest
import torch

from axonn_amd.optim import AdamW


def test_8_bit_moments_need_a_positive_eps_in_every_group():
    params = [torch.nn.Parameter(torch.zeros(8)) for _ in range(2)]
    for groups in ([dict(params=params[:1]), dict(params=params[1:], eps=0.0)], [dict(params=params, eps=0.0)],
                   [dict(params=params, eps=float("nan"))]):
        with pytest.raises(ValueError, match="positive epsilon"):
            AdamW(groups, state_bits=8)
        with pytest.raises(RuntimeError, match="GPU"):     # (fp32 moments take it, and then want a GPU)
            AdamW([{**group, "eps": 0.0} for group in groups], state_bits=32)
    with pytest.raises(RuntimeError, match="GPU"):
        AdamW([dict(params=params, eps=1e-6)], state_bits=8)
