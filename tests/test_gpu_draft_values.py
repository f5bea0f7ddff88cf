"""Values at the edges of drafted attention: scales far apart, rows a node does not see, scores that are no numbers, positions at the end of their range."""
import pytest
import torch

from tests import draft_cases as dc
from tests.test_gpu_draft import SCALE_CODE, dev, ints, run_attention
from zllm_amd import ops

pytestmark = pytest.mark.gpu

FORMS = [(torch.bfloat16, torch.bfloat16), (torch.float16, torch.float16), (torch.float32, torch.float32)]


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


@pytest.mark.parametrize("scales,large", [(torch.float16, 60000.0), (torch.bfloat16, 2.0**20), (torch.bfloat16, 2.0**60), (torch.bfloat16, 2.0**127), (torch.float32, 2.0**60),
                                          (torch.float32, 3.4e38)])
@pytest.mark.parametrize("q_dtype,out_dtype", FORMS + [(torch.bfloat16, torch.float32)])
@pytest.mark.parametrize("d,rows,kind", [(128, 6, "chain"), (192, 6, "chain"), (64, 40, "tree")])
def test_finite_scales_of_tokens_that_only_earlier_rows_see(scales, large, q_dtype, out_dtype, d, rows, kind):
    """The first tokens in reach of a window are seen by node 0 alone; their scales are the largest a cache holds.  The other rows stay within their bound."""
    c = dc.attention_case(10, [1000], rows, 8, 2, d, kind=kind, window=700, q_dtype=q_dtype, scales=scales)
    want, about = dc.attention(c, d**-0.5)
    bound = dc.attention_bound(c, want, about, out_dtype, out_dtype != torch.bfloat16 or q_dtype == torch.float32)
    others = c["positions"][0] > 1000
    slot = dc.physical(c["tables"], 0, [1000 + 1 - 700], c["page"])
    for sign in (1.0, -1.0):
        other = dict(c, v_scales=c["v_scales"].clone(), k_scales=c["k_scales"].clone())
        other["v_scales"][slot] = large * sign
        for k_large in (False, True):
            if k_large:
                other["k_scales"][slot] = large
            got = run_attention(other, d**-0.5, out_dtype).double().cpu()
            assert ((got - want).abs() <= bound)[others].all()
        if out_dtype != torch.float16 and large < 2.0**100:  # the row that sees them, as far as its type holds it
            other["k_scales"] = c["k_scales"]
            other["v_values"] = c["v_values"].clone()
            other["v_values"][slot] = other["v"][slot].double() * other["v_scales"][slot].double().repeat_interleave(64, -1)
            own, own_about = dc.attention(other, d**-0.5)
            own_bound = dc.attention_bound(c, own, own_about, out_dtype, out_dtype != torch.bfloat16 or q_dtype == torch.float32)
            got = run_attention(other, d**-0.5, out_dtype).double().cpu()
            assert ((got - own).abs() <= own_bound).all()


@pytest.mark.parametrize("q_dtype,out_dtype", FORMS)
@pytest.mark.parametrize("d", [128, 256])
@pytest.mark.parametrize("rows", [8, 40])
def test_f16_rows_that_a_node_does_not_see_may_be_anything(q_dtype, out_dtype, d, rows):
    """Values that are no numbers in the K and V row of one leaf, and of the first token in a window's reach: rows that do not see them keep their bits, and those
    that do have no number in the dimensions where V has none."""
    c = dc.attention_case(9, [50], rows, 8, 2, d, fmt="f16", kind="star", q_dtype=q_dtype)
    want = run_attention(c, d**-0.5, out_dtype).view(rows, 8, d)
    slot = dc.physical(c["tables"], 0, [50 + 5], c["page"])
    keep = [i for i in range(rows) if i != 5]
    dims = [3, d - 1, d + 64]
    for bad in (float("nan"), float("inf"), -float("inf")):
        other = dict(c, v=c["v"].clone())
        other["v"][slot, dims] = bad
        got = run_attention(other, d**-0.5, out_dtype).view(rows, 8, d)
        assert torch.equal(got[keep], want[keep])
        number = torch.isfinite(got[5])
        assert not number[:4, [3, d - 1]].any() and not number[4:, 64].any()
        number[:4, [3, d - 1]], number[4:, 64] = True, True
        assert number.all()
        other = dict(other, k=c["k"].clone())
        other["k"][slot] = bad
        assert torch.equal(run_attention(other, d**-0.5, out_dtype).view(rows, 8, d)[keep], want[keep])
    c = dc.attention_case(9, [1000, 30], rows, 8, 2, d, fmt="f16", kind="tree", q_dtype=q_dtype, window=700, counts=[rows, rows - 3])
    want = run_attention(c, d**-0.5, out_dtype).view(2, rows, 8, d)
    slot = dc.physical(c["tables"], 0, [1000 + 1 - 700], c["page"])
    keep = (c["positions"][0] > 1000).cuda()
    for bad in (float("nan"), float("inf"), -float("inf")):
        other = dict(c, v=c["v"].clone(), k=c["k"].clone())
        other["v"][slot], other["k"][slot] = bad, bad
        got = run_attention(other, d**-0.5, out_dtype).view(2, rows, 8, d)
        assert torch.equal(got[0][keep], want[0][keep]) and torch.equal(got[1], want[1])
        assert not torch.isfinite(got[0, 0]).any()


@pytest.mark.parametrize("q_dtype,out_dtype", FORMS)
@pytest.mark.parametrize("fmt", ["q8", "f16"])
@pytest.mark.parametrize("softcap", [0.0, 30.0])
def test_scores_that_are_no_numbers(q_dtype, out_dtype, fmt, softcap):
    """A row that sees a K row that holds no number, or whose query holds none, gives none, with a soft cap too; the other rows keep their bits."""
    c = dc.attention_case(9, [50], 8, 8, 2, 128, fmt=fmt, kind="star", q_dtype=q_dtype)
    want = run_attention(c, 128**-0.5, out_dtype, softcap)
    slot = dc.physical(c["tables"], 0, [50 + 5], c["page"])
    name = "k_scales" if fmt == "q8" else "k"
    other = {**c, name: c[name].clone()}
    other[name][slot] = float("nan")
    other["q"] = c["q"].clone()
    other["q"][2] = float("nan")
    got = run_attention(other, 128**-0.5, out_dtype, softcap)
    keep = [0, 1, 3, 4, 6, 7]
    assert torch.equal(got[keep], want[keep])
    assert torch.isnan(got[[2, 5]]).all()
    cached = {**c, name: c[name].clone()}
    cached[name][dc.physical(c["tables"], 0, [7], c["page"])] = float("nan")
    assert torch.isnan(run_attention(cached, 128**-0.5, out_dtype, softcap)).all()


@pytest.mark.parametrize("window", [1, 40, 2**31 - 256])
def test_positions_at_the_end_of_their_range(window):
    """Nodes at 2^32 - 1 and just before it: a window that does not reach back to the cached tokens holds none of them."""
    c = dc.attention_case(11, [100, 37], 9, 8, 2, 128, window=window, kind="chain")
    c["positions"] = c["positions"].long()
    c["positions"][0] += 2**32 - 1 - 100 - 8
    c["positions"][1, 4:] = 2**32 - 1
    scale = 128**-0.5
    want, about = dc.attention(c, scale)
    for out_dtype in (torch.bfloat16, torch.float32):
        got = run_attention(c, scale, out_dtype, positions=dev(c["positions"].to(torch.int32))).double().cpu()
        assert ((got - want).abs() <= dc.attention_bound(c, want, about, out_dtype, out_dtype != torch.bfloat16)).all()



@pytest.mark.parametrize("gate_cols", [1, 8 * 128])
def test_gates_of_rows_that_give_zeros(gate_cols):
    """Nodes that are not there, and rows that see nothing, give zeros whatever their gates hold."""
    c = dc.attention_case(8, [0, 90], 5, 8, 2, 128, counts=[3, 2], empty=[(0, 1)])
    gate = torch.zeros(10, gate_cols)
    want = run_attention(c, 128**-0.5, torch.bfloat16, gate=dev(gate))
    zeros = [1, 3, 4, 7, 8, 9]
    for bad in (float("nan"), float("inf"), -float("inf")):
        gate[zeros] = bad
        got = run_attention(c, 128**-0.5, torch.bfloat16, gate=dev(gate))
        assert torch.equal(got, want) and (got[zeros] == 0).all()



@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads", [4, 20, 50])
@pytest.mark.parametrize("power", [40, 70, 110])
def test_large_scales_behind_scales_of_zero(out_dtype, heads, power):
    """V rows of zeros (a stored scale of zero), then one row with a scale of 2^power, in one part: the rows of zeros keep their share of the normaliser."""
    n, page = 320, 16
    c = dc.attention_case(3, [n], 2, heads, 1, 128, scales=torch.bfloat16)
    last = dc.physical(c["tables"], 0, [n - 1], page)
    c["k_scales"].fill_(2.0**-20)
    c["v_scales"].fill_(0.0)
    c["v_scales"][last] = 2.0**power
    c["v"][last] = 100
    for name in ("k", "v"):
        c[name][c[name] == -128] = 0
        c[name + "_values"] = (c[name].view(-1, 2, 64).double() * c[name + "_scales"].double()[..., None]).view(c[name].shape)
    want, about = dc.attention(c, 128**-0.5)
    got = ops.gqa_draft_attention(dev(c["q"]), dev(c["k"]), dev(c["k_scales"]), dev(c["v"]), dev(c["v_scales"]), dev(c["tables"]), ints([n]), dev(c["masks"]), heads, 1, 128,
                                  page, 128**-0.5, 0, scale_dtype=SCALE_CODE[torch.bfloat16], out_dtype=out_dtype).double().cpu()
    assert ((got - want).abs() <= dc.attention_bound(c, want, about, out_dtype, out_dtype != torch.bfloat16)).all()



@pytest.mark.parametrize("q_dtype,out_dtype", [(torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32), (torch.float32, torch.float32)])
@pytest.mark.parametrize("heads", [4, 20, 50])
@pytest.mark.parametrize("power", [24, 30, 60, 100, 122])
def test_scores_far_from_zero(q_dtype, out_dtype, heads, power):
    """Queries up to the end of their range: scores are numbers, and so are the outputs, those of the largest score alone."""
    c = dc.attention_case(11, [200], 6, heads, 1, 128, q_dtype=q_dtype)
    about = dc.attention(c, 128**-0.5)[1]
    c["q"][2] *= 2.0**power
    got = run_attention(c, 128**-0.5, out_dtype).double().cpu()
    right, _ = dc.attention(c, 128**-0.5)
    keep = [0, 1, 3, 4, 5]
    assert ((got - right).abs() <= dc.attention_bound(c, right, about, out_dtype, out_dtype != torch.bfloat16 or q_dtype == torch.float32))[keep].all()
    half = dc.EPS[out_dtype] + 2.0**-9  # the output's rounding; probabilities and V rows as f16
    assert ((got[2] - right[2]).abs() <= half * right[2].abs() + 2.0**-20).all()
