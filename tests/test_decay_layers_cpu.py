"""What nn.DecayAttention refuses before any device work."""
import pytest
import torch
import torch.nn as nn


@pytest.mark.parametrize("sizes,heads,kv_heads", [((64, 31, 33), 2, 2), ((64, 32, 33), 2, 2), ((65, 32, 32), 2, 2),
                                                  ((64, 64, 32), 4, 2), ((64, 64, 64), 0, 1), ((64, 64, 64), 2, 0)])
def test_layers_that_do_not_divide_into_heads(sizes, heads, kv_heads):
    """Also where the sizes add up all the same: 31 + 33 columns are not two keys and two values of 16."""
    from snn_compiler.nn import DecayAttention
    q, k, v = (nn.Linear(96, n) for n in sizes)
    with pytest.raises(ValueError, match="heads"):
        DecayAttention.from_linears(q, k, v, nn.Linear(32, 96), torch.ones(max(heads, 1)), heads=heads,
                                    kv_heads=kv_heads)
