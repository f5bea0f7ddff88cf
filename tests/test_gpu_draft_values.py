"""Values at the edges of drafted attention: scales far apart, rows a node does not see, scores that are no numbers, positions at the end of their range."""
import pytest
import torch

from tests import draft_cases as dc
from tests.test_gpu_draft import SCALE_CODE, dev, ints
from zllm_amd import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("lag", [1, 3, 8, 12, 16, 20, 40, 120])
@pytest.mark.parametrize("scales", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads", [4, 20, 50])
def test_tokens_whose_scales_lie_far_below_the_first_ones(lag, scales, heads):
    """One token of weight near 1 with a large V scale, then 32,768 of 2^-20 each, their V scales 2^lag lower, in one part (an estimate of no tokens): together
    they are 3 % of the normaliser, whatever the scales of their values are.  One, two and four waves of pairs."""
    n, page = 32768, 16
    c = dc.attention_case(lag, [n], 2, heads, 1, 128, scales=scales)
    first = dc.physical(c["tables"], 0, [0], page)
    gen = torch.Generator().manual_seed(lag)
    for name in ("k", "v"):
        c[name] = torch.randint(-127, 128, c[name].shape, generator=gen, dtype=torch.int8)
        c[name + "_scales"].fill_(2.0**-20 if name == "k" else 2.0**-lag)
    c["k"][first], c["k_scales"][first] = 127, 13.9 * 128**0.5 / (128 * 127)
    c["v_scales"][first] = 1.0
    for name in ("k", "v"):
        c[name + "_values"] = (c[name].view(-1, 2, 64).double() * c[name + "_scales"].double()[..., None]).view(c[name].shape)
    c["q"].fill_(1.0)
    one = dict(c, hq=1, q=c["q"][:, :128].contiguous())  # all heads are alike
    want, about = dc.attention(one, 128**-0.5)
    bound = dc.attention_bound(one, want, about, torch.bfloat16, False)
    got = ops.gqa_draft_attention(dev(c["q"]), dev(c["k"]), dev(c["k_scales"]), dev(c["v"]), dev(c["v_scales"]), dev(c["tables"]), ints([n]), dev(c["masks"]), heads, 1, 128,
                                  page, 128**-0.5, 0, scale_dtype=SCALE_CODE[scales], out_dtype=torch.bfloat16).double().cpu()
    assert ((got.view(2, heads, 128) - want.view(2, 1, 128)).abs() <= bound.view(2, 1, 128)).all()
