"""expert_mlp's kernels where a workgroup goes on to further columns, takes two groups of them, or has 16 columns of the result:
against the definition in 64 bits."""

import pytest
import torch

import adambridge_amd as ab
from test_expert_mlp_gpu import BF16, FP32, _check, _operands

pytestmark = pytest.mark.gpu


# chosen experts times columns of 16 pass the 1024 workgroups once, in one group of columns (3500, 3501) and in two (4200 and
# more); 8200 of 16 experts four times; an expert's last columns are a part of a group, and of two
@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("hidden", [40, 41])
@pytest.mark.parametrize("tokens,experts,inter", [(13, 8, 3500), (13, 8, 3501), (13, 8, 4200), (13, 8, 4209), (16, 16, 8200), (16, 16, 8211)])
@pytest.mark.parametrize("gated,activation,normalize", [(False, "gelu", True), (True, "silu", False)])
def test_more_columns_than_workgroups(tokens, experts, inter, hidden, gated, activation, normalize, dtype):
    gen = torch.Generator("cuda").manual_seed(inter + hidden)
    _check(tokens, experts, 2, inter, hidden, dtype, gated, activation, normalize, gen)


# up's sums of many steps there: the next columns' first weights are asked for in the last one
@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("inter,hidden", [(4200, 1000), (4209, 1003), (3501, 515)])
def test_more_columns_than_workgroups_of_long_rows(inter, hidden, gated, dtype):
    gen = torch.Generator("cuda").manual_seed(inter + hidden)
    _check(13, 8, 2, inter, hidden, dtype, gated, "gelu", True, gen)


# 4, 8 and 16 columns of the result a workgroup, and sizes about the steps between them
@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("inter", [24, 33, 1030])
@pytest.mark.parametrize("hidden", [1024, 1025, 1536, 2047, 2048, 2049, 2051, 4095, 4096, 4101, 4104, 5000])
def test_columns_of_the_result(hidden, inter, gated, dtype):
    gen = torch.Generator("cuda").manual_seed(inter + hidden)
    _check(7, 5, 3, inter, hidden, dtype, gated, "silu", True, gen)


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("inter,hidden", [(4200, 40), (3501, 41), (40, 4101)])
def test_what_an_expert_holds_stays_with_its_tokens(inter, hidden, dtype):
    gen = torch.Generator("cuda").manual_seed(2)
    x, logits, up, down, gate = _operands(10, 8, inter, hidden, dtype, True, gen)
    clean = ab.expert_mlp(x, logits, up, down, 2, gate)
    chose = (ab.route(logits, 2).experts == 3).any(1)
    assert 0 < chose.sum() < 10
    for poisoned in (up, gate, down):
        kept = poisoned[3].clone()
        poisoned[3] = torch.nan
        got = ab.expert_mlp(x, logits, up, down, 2, gate)
        assert torch.equal(got[~chose], clean[~chose]) and got[chose].isnan().all()
        poisoned[3] = kept
    x[4] = torch.inf
    others = torch.arange(10, device="cuda") != 4
    assert torch.equal(ab.expert_mlp(x, logits, up, down, 2, gate)[others], clean[others])
