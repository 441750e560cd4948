"""Adapters at the edges of their formula: scales of adapters that no token names, and the backward pass of few tokens whose
long axis is shared by several workgroups.  Tolerances as in test_gpu_lora."""
import math

import pytest
import torch

from test_gpu_dense import PAIRS, TYPES, rand
from test_gpu_lora import adapters, check_backward, some_ids

pytestmark = pytest.mark.gpu


# ids of one slice of tokens for each adapter, and of several (few columns and more than 512 tokens)
@pytest.mark.parametrize("xt,wt", [("f32", "f32"), ("bf16", "bf16")])
@pytest.mark.parametrize("S,I,O,R", [(3, 72, 40, 5), (700, 264, 520, 16), (6000, 128, 96, 24), (40, 300, 8192, 65)])
def test_scale_of_an_adapter_without_tokens(S, I, O, R, xt, wt):
    """Nothing reads it: zeros for its gradients, and all other results as with a scale of 1 in its place."""
    import zeromoe_amd as Z

    n = 5
    a, b = adapters(n, R, I, O, wt)
    x, dy, v = rand(S, I, seed=3, dtype=TYPES[xt]), rand(S, O, seed=4, dtype=TYPES[xt]), rand(S, R, seed=5)
    ids = torch.tensor([1, 3], device="cuda", dtype=torch.int32)[some_ids(S, 2, "runs").long()]
    scale = rand(n, seed=6)
    scale[0], scale[2], scale[4] = math.inf, math.nan, -math.inf
    good = scale.nan_to_num(1.0, 1.0, 1.0)
    got = (Z.lora(x, a, b, ids, scale=scale), *Z.lora_backward(dy, x, a, b, ids, v, scale=scale))
    want = (Z.lora(x, a, b, ids, scale=good), *Z.lora_backward(dy, x, a, b, ids, v, scale=good))
    for g, w in zip(got, want):
        assert torch.equal(g, w)
    for g in got[2:]:
        assert (g[[0, 2, 4]] == 0).all()


# O of several slices in the backward pass, ranks of each kind of kernel, odd sizes
SPLIT = [(1, 520, 8200, 128, 3), (63, 300, 8192, 65, 1), (40, 260, 4099, 200, 3), (5, 1030, 4608, 30, 2), (2, 2100, 8191, 16, 1),
         (100, 131, 5121, 100, 4)]


@pytest.mark.parametrize("xt,wt", PAIRS)
@pytest.mark.parametrize("S,I,O,R,n", SPLIT)
def test_backward_of_few_tokens_and_a_long_axis(S, I, O, R, n, xt, wt):
    for need in ((True, True, True), (True, False, False), (False, True, False)):
        check_backward(S, I, O, R, n, xt, wt, need=need)
    check_backward(S, I, O, R, n, xt, wt, "one", ydt="f32", seed=21)
