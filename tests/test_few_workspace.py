"""What the layer for a few tokens asks of the workspace: nothing that moe_forward_static's array has no room for."""
import pytest
import torch

import cuplayground_amd as moe
from cuplayground_amd import api

STATIC = 32 << 20                    # MOE355_STATIC_WORKSPACE_BYTES


def _config(S, H, I, E, k, dtype=api.DTYPE_BF16):
    return moe.MoEConfig(expert_top_k=k, hidden_size=H, intermediate_size=I, micro_batch=1, num_experts=E, sequence_len=S, torch_dtype=dtype)


# What the layers took before there was a layer for a few tokens, just under the array's size: with the experts' output rows larger than
# the shared sums of 16 columns (the first) and smaller.
NEAR = [(16, 1024, 64000, 16, 16, 33383680), (16, 64, 64000, 512, 16, 33385728), (1, 1024, 1044864, 16, 16, 33553408), (4, 512, 260928, 16, 16, 33549312),
        (16, 2048, 520832, 16, 2, 33551872), (16, 1024, 1044800, 16, 1, 33552896)]


@pytest.mark.parametrize("dtype", [api.DTYPE_BF16, api.DTYPE_FP16])
@pytest.mark.parametrize("S,H,I,E,k,before", NEAR)
def test_layers_that_fitted_the_static_workspace_fit_it(S, H, I, E, k, before, dtype):
    assert before <= STATIC
    assert _config(S, H, I, E, k, dtype).workspace_bytes() == before


def test_workspace_of_layers_that_have_no_shared_sums_or_rows_enough():
    """e4m3 layers, 17 tokens, wide layers: as before; and where the experts' output rows hold the sums."""
    for S, H, I, E, k, dtype, before in ((16, 1024, 4096, 8, 2, api.DTYPE_FP8, 405760), (3, 128, 128, 8, 2, api.DTYPE_FP8, 80640),
                                         (16, 2048, 1408, 64, 6, api.DTYPE_BF16, 800512)):
        assert _config(S, H, I, E, k, dtype).workspace_bytes() == before


@pytest.mark.gpu
@pytest.mark.parametrize("S,H,I,E,k", [(16, 1024, 64000, 16, 16), (16, 1024, 520832, 2, 2)])
def test_such_layers_run_on_the_static_workspace_and_for_a_few_tokens(S, H, I, E, k):
    """The two largest of their kind: moe_forward_static is moe_forward to the bit; the layer for a few tokens differs by the rounding of the
    experts' rows, 2^-8 of each, that it does not make, and both round the intermediate and the output: four half units of all values together."""
    g = torch.Generator(device="cuda").manual_seed(S + E)

    def normal(*shape, std):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.bfloat16) * std

    w = {"gate_w": normal(E, H, std=0.05), "w_up": normal(E, I, H, std=H ** -0.5), "w_down": normal(E, H, I, std=I ** -0.5)}
    x = normal(S, H, std=1.0)
    layer = moe.MoELayer(_config(S, H, I, E, k))
    want = layer.forward(x, w)
    assert torch.equal(layer.forward(x, w, static_workspace=True), want)
    got = layer.forward_few(x, w)
    assert torch.equal(layer.forward_few(x, w), got)
    assert (got.double() - want.double()).norm() <= 4 * 2.0 ** -8 * want.double().norm()
