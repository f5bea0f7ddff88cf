"""The drafted-token operators on the device: against their definitions in 64 bits, against the operators that exist for one sequence, in a run
together, captured and replayed."""
import pytest
import torch

from tests import draft_cases as dc
from zllm_amd import capi, ops

pytestmark = pytest.mark.gpu

SCALE_CODE = {torch.bfloat16: capi.SCALE_BF16, torch.float16: capi.SCALE_F16, torch.float32: capi.SCALE_F32}


def dev(t):
    return None if t is None else t.to("cuda")


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


# ---- layout --------------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("kind", ["chain", "tree", "star", "forest"])
@pytest.mark.parametrize("batch,rows", [(1, 1), (3, 2), (2, 63), (2, 64), (5, 65), (1, 130), (3, 256)])
def test_layout(kind, batch, rows):
    gen = torch.Generator().manual_seed(rows)
    parents = dc.tree(gen, batch, rows, kind)
    counts = [rows - (b * 7) % (rows + 1) for b in range(batch)]
    lens = [1000 * b + b for b in range(batch)]
    sees, depth = dc.ancestors(parents, counts)
    masks, positions = ops.draft_layout(dev(parents), ints(lens), row_counts=ints(counts))
    assert torch.equal(masks.cpu(), dc.pack(sees))
    assert torch.equal(positions.cpu(), torch.tensor(lens, dtype=torch.int32)[:, None] + depth)
    if batch == 3:
        sees, depth = dc.ancestors(parents, [rows] * batch)
        assert torch.equal(ops.draft_layout(dev(parents), ints(lens))[0].cpu(), dc.pack(sees))


# ---- prologue ------------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("hq,hkv,d,rotary,half,rule,src,q_out", [
    (8, 2, 128, 128, True, capi.QUANT_METAL_GQA, torch.bfloat16, torch.bfloat16),
    (4, 4, 64, 32, False, capi.QUANT_ROCM_MLA, torch.float32, torch.float32),
    (6, 2, 256, 64, True, capi.QUANT_CUDA_GQA, torch.float16, torch.float32),
    (3, 1, 192, 192, False, capi.QUANT_METAL_GQA, torch.bfloat16, torch.float32),
    (2, 2, 128, 0, True, capi.QUANT_METAL_GQA, torch.bfloat16, torch.bfloat16),
])
@pytest.mark.parametrize("cache", ["q8", "f16"])
def test_prologue_rows_equal_those_of_single_rows(hq, hkv, d, rotary, half, rule, src, q_out, cache):
    """Every node's row has the bits of gqa_prologue called for that row alone; everything else in the planes stays."""
    gen = torch.Generator().manual_seed(d + rotary)
    batch, rows, page = 3, 5, 8
    lens, counts = [0, 13, 30], [5, 3, 4]
    parents = dc.tree(gen, batch, rows, "tree")
    _, depth = dc.ancestors(parents, [rows] * batch)
    positions = torch.tensor(lens, dtype=torch.int32)[:, None] + depth
    tables, pool = dc.block_tables(gen, [n + rows for n in lens], page)
    cols = hkv * d
    q, k, v = (torch.randn(batch * rows, h * d, generator=gen).to(src).cuda() for h in (hq, hkv, hkv))
    q_norm, k_norm = (torch.randn(d, generator=gen).cuda() * 0.2 for _ in range(2))
    angle = torch.rand(64, max(rotary // 2, 1), generator=gen) * 6.0
    cos, sin = (angle.cos().cuda(), angle.sin().cuda()) if rotary else (None, None)
    f16 = cache == "f16"
    scale_type = {capi.QUANT_METAL_GQA: torch.float16, capi.QUANT_ROCM_MLA: torch.bfloat16, capi.QUANT_CUDA_GQA: torch.float32}[rule]

    def planes(n):
        if f16:
            return [torch.full((n, cols), 7.0, dtype=torch.float16, device="cuda"), None] * 2
        return [torch.full((n, cols), 99, dtype=torch.int8, device="cuda"), torch.full((n, cols // 64), 5.0, dtype=scale_type, device="cuda")] + [
            torch.full((n, cols), 99, dtype=torch.int8, device="cuda"), torch.full((n, cols // 64), 5.0, dtype=scale_type, device="cuda")]

    if f16:
        kp, vp = planes(pool)[0], planes(pool)[0]
        got_planes = [kp, None, vp, None]
    else:
        got_planes = planes(pool)
    want_planes = [None if t is None else t.clone() for t in got_planes]
    got = ops.gqa_draft_prologue(q, k, v, q_norm, k_norm, cos, sin, *got_planes, dev(tables), ints(lens), hq, hkv, d, rotary, page, positions=dev(positions),
                                 row_counts=ints(counts), rule=rule, split_half=half, q_out_dtype=q_out, kv_format=capi.KV_F16 if f16 else capi.KV_Q8G64)
    want = torch.zeros_like(got)
    for b in range(batch):
        for i in range(counts[b]):
            r, at = b * rows + i, int(positions[b, i])
            single = [torch.zeros(64, cols, dtype=torch.int8, device="cuda"), torch.zeros(64, cols // 64, dtype=scale_type, device="cuda")]
            single += [t.clone() for t in single]
            args = (cos, sin, *single, None, at)
            want[r] = ops.gqa_prologue(q[r : r + 1], k[r : r + 1], v[r : r + 1], q_norm, k_norm, *args, hq, hkv, d, rotary, page, rule=rule, split_half=half,
                                       q_out_dtype=q_out)[0]
            slot = int(dc.physical(tables, b, [lens[b] + i], page)[0])
            if f16:
                as_query = ops.gqa_prologue(k[r : r + 1], k[r : r + 1], v[r : r + 1], k_norm, k_norm, *args, hkv, hkv, d, rotary, page, rule=rule, split_half=half)
                want_planes[0][slot], want_planes[2][slot] = as_query[0].half(), v[r].half()
            else:
                for plane, one in zip(want_planes, single):
                    plane[slot] = one[at]
    assert torch.equal(got.view(torch.int16 if q_out != torch.float32 else torch.int32), want.view(torch.int16 if q_out != torch.float32 else torch.int32))
    for one, other in zip(got_planes, want_planes):
        assert one is None or torch.equal(one, other)
    if f16 and q_out == torch.float32:
        as_f16 = ops.gqa_draft_prologue(q, k, v, q_norm, k_norm, cos, sin, *got_planes, dev(tables), ints(lens), hq, hkv, d, rotary, page,
                                        positions=dev(positions), row_counts=ints(counts), split_half=half, q_out_dtype=torch.float16, kv_format=capi.KV_F16)
        assert torch.equal(as_f16, want.half())


def test_prologue_chain_ring_and_unaligned():
    """No positions: a chain behind each sequence's tokens; a ring's slots; tensors that are not 16-byte aligned; nodes behind the pages."""
    gen = torch.Generator().manual_seed(5)
    batch, rows, d, page = 2, 4, 64, 4
    lens = [9, 21]
    q, k, v = (torch.randn(batch * rows, d, generator=gen).cuda() for _ in range(3))
    angle = torch.rand(26, 32, generator=gen)
    cos, sin = angle.cos().cuda(), angle.sin().cuda()
    outs = []
    for shift in (0, 1):
        codes = [torch.zeros(24 * d + 16, dtype=torch.int8, device="cuda")[shift : 24 * d + shift].view(24, d) for _ in range(2)]
        steps = [torch.zeros(24, 1, dtype=torch.float16, device="cuda") for _ in range(2)]
        tables = torch.tensor([[0, 1, 2], [5, 4, 3]], dtype=torch.int32)
        got = ops.gqa_draft_prologue(q, k, v, None, None, cos, sin, codes[0], steps[0], codes[1], steps[1], dev(tables), ints(lens), 1, 1, d, d, page, ring_capacity=12)
        outs.append((got, codes, steps))
        for b in range(batch):
            for i in range(rows):
                slot = int(dc.physical(tables, b, [lens[b] + i], page, 12)[0])
                single = [torch.zeros(26, d, dtype=torch.int8, device="cuda"), torch.zeros(26, 1, dtype=torch.float16, device="cuda")]
                single += [t.clone() for t in single]
                r = b * rows + i
                want = ops.gqa_prologue(q[r : r + 1], k[r : r + 1], v[r : r + 1], None, None, cos, sin, *single, None, lens[b] + i, 1, 1, d, d, page)
                assert torch.equal(got[r], want[0])
                assert torch.equal(codes[0][slot], single[0][lens[b] + i]) and torch.equal(steps[1][slot], single[3][lens[b] + i])
    assert torch.equal(outs[0][1][1], outs[1][1][1])
    # sequence 1's nodes 3 .. lie behind its six pages: not written; the position past the tables takes their last row
    codes = [torch.zeros(24, d, dtype=torch.int8, device="cuda") for _ in range(2)]
    steps = [torch.zeros(24, 1, dtype=torch.float16, device="cuda") for _ in range(2)]
    tables = torch.zeros(2, 6, dtype=torch.int32)
    tables[0], tables[1] = torch.arange(6), 5
    ops.gqa_draft_prologue(q, k, v, None, None, cos[:20], sin[:20], codes[0], steps[0], codes[1], steps[1], dev(tables), ints([9, 22]), 1, 1, d, d, page)
    assert int((steps[0][:, 0] != 0).sum()) == 4 + 2  # slots 9 .. 12, and 22, 23 of sequence 1 in page 5


@pytest.mark.parametrize("d", [64, 128, 192])
def test_prologue_reciprocal_rule(d):
    """Bit for bit the rows that a tensor program writes whose constants divide as products with reciprocals; ties of codes among them."""
    gen = torch.Generator().manual_seed(d)
    nodes, heads, page = 200, 2, 16
    x = torch.randn(3, nodes, heads * d, generator=gen).bfloat16()
    x[2] = torch.where(torch.rand(nodes, heads * d, generator=gen) < 0.5, torch.randint(-254, 255, (nodes, heads * d), generator=gen) * 0.5, 0.0).bfloat16()
    x[2].view(-1, 64)[:, 0] = 127.0  # a scale of one, and codes half way between two
    q, k, v = x.cuda()
    norm = (torch.randn(d, generator=gen) * 0.1).cuda()
    tables = torch.randperm(nodes // 8, generator=gen).to(torch.int32).view(25, 1)
    planes = [torch.zeros(25 * page, heads * d, dtype=torch.int8, device="cuda"), torch.zeros(25 * page, heads * d // 64, dtype=torch.float16, device="cuda")]
    planes += [t.clone() for t in planes]
    got = ops.gqa_draft_prologue(q, k, v, norm, norm, None, None, *planes, dev(tables), ints([0] * 25), heads, heads, d, 0, page, rule=capi.QUANT_RECIPROCAL_GQA)

    def normed(t):
        t = t.float().view(nodes, heads, d)
        total = torch.zeros(nodes, heads, 8, device="cuda")
        for c in range(d // 8):
            total = total + t[..., 8 * c : 8 * c + 8] * t[..., 8 * c : 8 * c + 8]
        total = total[..., :4] + total[..., 4:]
        total = total[..., :2] + total[..., 2:]
        total = total[..., :1] + total[..., 1:]
        mean = total * torch.tensor(1.0 / d, dtype=torch.float32, device="cuda")
        return t * (torch.ones_like(mean) / torch.sqrt(mean + torch.tensor(1e-6, device="cuda"))) * (norm + 1.0)

    assert torch.equal(got.view(nodes, heads, d), normed(q))
    rows = (tables.long() * page + torch.arange(8)).flatten().cuda()
    for t, codes, steps in ((normed(k), planes[0], planes[1]), (v.float(), planes[2], planes[3])):
        groups = t.reshape(nodes, -1, 64)
        step = groups.abs().amax(-1) * torch.tensor(1.0 / 127.0, dtype=torch.float32, device="cuda")
        assert torch.equal(steps[rows], step.half())
        assert torch.equal(codes[rows].view(nodes, -1, 64), torch.round(groups * (torch.ones_like(step) / step)[..., None]).clamp(-127, 127).to(torch.int8))


# ---- attention -----------------------------------------------------------------------------------------------------------


def run_attention(c, scale, out_dtype, softcap=0.0, gate=None, total=True, chain=False, **more):
    kw = dict(positions=dev(c["positions"]), row_counts=ints(c["counts"]), window=c["window"], softcap=softcap, ring_capacity=c["ring"], out_dtype=out_dtype, gate=gate,
              kv_format=capi.KV_F16 if c["fmt"] == "f16" else capi.KV_Q8G64, total_kv_tokens=sum(c["lens"]) if total else 0)
    if c["fmt"] != "f16":
        kw["scale_dtype"] = SCALE_CODE[c["k_scales"].dtype]
    kw.update(more)
    return ops.gqa_draft_attention(dev(c["q"]), dev(c["k"]), dev(c["k_scales"]), dev(c["v"]), dev(c["v_scales"]), dev(c["tables"]), ints(c["lens"]),
                                   None if chain else dev(c["masks"]), c["hq"], c["hkv"], c["d"], c["page"], scale, max(c["lens"]), **kw)


def check_attention(c, out_dtype, softcap=0.0, gate=None, scale=None, **more):
    scale = c["d"] ** -0.5 if scale is None else scale
    got = run_attention(c, scale, out_dtype, softcap, dev(gate), **more).double().cpu()
    want, about = dc.attention(c, scale, softcap, gate)
    exact = out_dtype != torch.bfloat16 or c["q"].dtype == torch.float32
    bound = dc.attention_bound(c, want, about, out_dtype, exact, softcap)
    off = (got - want).abs()
    assert torch.isfinite(got).all()
    assert (off <= bound).all(), f"{float((off - bound).max()):.3e} over, at most {float((off / bound.clamp(min=1e-30)).max()):.2f} of the bound"
    return got, want


SHAPES = [  # lens, rows, heads, dim
    ([0], 1, (1, 1), 64), ([1], 1, (4, 4), 128), ([31], 2, (8, 1), 128), ([32], 3, (6, 2), 128), ([33, 0, 700], 5, (16, 4), 128),
    ([500, 64], 7, (8, 2), 64), ([95], 33, (5, 1), 192), ([300, 17], 12, (16, 8), 256), ([1500], 64, (8, 1), 128), ([130], 100, (3, 1), 128),
    ([40], 256, (2, 2), 64), ([257, 1], 20, (12, 2), 192), ([2049], 9, (64, 8), 128),
]


@pytest.mark.parametrize("lens,rows,heads,d", SHAPES)
@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float32])
def test_attention_q8(lens, rows, heads, d, out_dtype):
    check_attention(dc.attention_case(rows + d, lens, rows, *heads, d), out_dtype)


@pytest.mark.parametrize("lens,rows,heads,d", [s for s in SHAPES if s[3] in (128, 256)])
@pytest.mark.parametrize("q_dtype,out_dtype", [(torch.float16, torch.float16), (torch.float32, torch.bfloat16)])
def test_attention_f16_rows(lens, rows, heads, d, q_dtype, out_dtype):
    check_attention(dc.attention_case(rows + d, lens, rows, *heads, d, fmt="f16", q_dtype=q_dtype), out_dtype)


@pytest.mark.parametrize("scales", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("q_dtype,out_dtype", [(torch.bfloat16, torch.float16), (torch.float32, torch.float32), (torch.float16, torch.bfloat16)])
@pytest.mark.parametrize("d", [64, 128, 192, 256])
def test_attention_types(scales, q_dtype, out_dtype, d):
    check_attention(dc.attention_case(3, [77, 200], 6, 8, 2, d, scales=scales, q_dtype=q_dtype, kind="forest"), out_dtype)


@pytest.mark.parametrize("rows,heads", [(10, (8, 2)), (25, (8, 2)), (2, (256, 1)), (256, (8, 1))])
@pytest.mark.parametrize("fmt,d", [("q8", 64), ("q8", 128), ("q8", 192), ("q8", 256), ("f16", 128), ("f16", 256)])
def test_attention_pairs(rows, heads, fmt, d):
    """Pairs that fill one, two or four waves, and many tiles of them; every form."""
    c = dc.attention_case(rows, [333, 5] if rows < 256 else [70], rows, *heads, d, fmt=fmt)
    check_attention(c, torch.bfloat16)
    check_attention(c, torch.float16)
    check_attention(dict(c, q=c["q"].float()), torch.float32)


@pytest.mark.parametrize("total", [True, False])
def test_attention_many_sequences(total):
    """More sequences than lanes, some without nodes: parts are numbered over all of them."""
    lens = [(b * 37) % 150 for b in range(150)]
    counts = [(b * 5) % 4 for b in range(150)]
    c = dc.attention_case(12, lens, 3, 2, 1, 64, counts=counts)
    check_attention(c, torch.bfloat16, total=total)


@pytest.mark.parametrize("page", [1, 5, 24, 64, 1000])
@pytest.mark.parametrize("rows", [4, 40])
def test_attention_pages(page, rows):
    check_attention(dc.attention_case(page, [150, 3], rows, 8, 2, 128, page=page), torch.bfloat16)


@pytest.mark.parametrize("window,lens", [(1, [50]), (7, [3, 100]), (64, [64, 63, 500]), (300, [700])])
@pytest.mark.parametrize("fmt,d", [("q8", 128), ("f16", 256)])
@pytest.mark.parametrize("softcap", [0.0, 30.0])
def test_attention_window(window, lens, fmt, d, softcap):
    """A window of one: a node sees itself; windows shorter than the tree; rows in front of the window hold no numbers."""
    c = dc.attention_case(window, lens, 11, 8, 2, d, fmt=fmt, window=window)
    check_attention(c, torch.bfloat16, softcap)
    check_attention(c, torch.float32, softcap)


def test_attention_ring():
    for lens in ([10, 200], [95]):
        check_attention(dc.attention_case(1, lens, 6, 8, 2, 128, window=32, ring=40, page=8), torch.bfloat16)


def test_attention_chain_needs_no_masks():
    c = dc.attention_case(2, [100, 40], 70, 4, 2, 128, kind="chain", counts=[70, 33])
    got, _ = check_attention(c, torch.bfloat16)
    assert torch.equal(run_attention(c, 128**-0.5, torch.bfloat16, chain=True).double().cpu(), got)


@pytest.mark.parametrize("softcap,scale", [(50.0, 0.088), (5.0, 1.0), (1000.0, 0.088)])
@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float32])
def test_attention_soft_cap(softcap, scale, out_dtype):
    check_attention(dc.attention_case(4, [300], 10, 8, 2, 128), out_dtype, softcap, scale=scale)


def test_attention_gate():
    c = dc.attention_case(6, [90, 20], 5, 8, 2, 128, counts=[5, 2])
    gen = torch.Generator().manual_seed(1)
    for gate in (torch.randn(10, 1, generator=gen), torch.randn(10, 8 * 128, generator=gen).bfloat16()):
        got = run_attention(c, 128**-0.5, torch.float32, gate=dev(gate)).double().cpu()
        want, about = dc.attention(c, 128**-0.5, 0.0, gate)
        # the gate's own exponential and division: 2^-21 of the value
        assert ((got - want).abs() <= dc.attention_bound(c, want, about, torch.float32, True) + 2.0**-21 * about[0]).all()


@pytest.mark.parametrize("fmt", ["q8", "f16"])
def test_attention_rows_that_see_nothing(fmt):
    """No cached token and an empty mask: zeros.  Nodes that are not there: zeros, their queries may be anything.  A sequence without nodes."""
    c = dc.attention_case(8, [0, 0, 40], 6, 8, 2, 128, fmt=fmt, counts=[6, 4, 0], empty=[(0, 0), (0, 3), (1, 1)])
    c["q"].view(3, 6, -1)[1, 4:] = float("inf")
    c["q"].view(3, 6, -1)[2] = float("nan")
    got, _ = check_attention(c, torch.bfloat16)
    zero = got.view(3, 6, -1)
    assert (zero[0, 0] == 0).all() and (zero[0, 3] == 0).all() and (zero[1, 1] == 0).all() and (zero[1, 4:] == 0).all() and (zero[2] == 0).all()
    assert (zero[0, 1] != 0).any()


def test_attention_what_a_node_does_not_see_may_be_anything():
    """A node whose scales are not numbers or infinite, seen by one leaf only: every other row keeps the bits it has with an ordinary node there."""
    c = dc.attention_case(9, [50], 8, 8, 2, 128, kind="star")
    want = run_attention(c, 128**-0.5, torch.bfloat16)
    slot = dc.physical(c["tables"], 0, [50 + 5], c["page"])
    for bad in (float("nan"), float("inf"), 60000.0):
        other = dict(c, k_scales=c["k_scales"].clone(), v_scales=c["v_scales"].clone())
        other["k_scales"][slot] = bad
        other["v_scales"][slot] = bad
        got = run_attention(other, 128**-0.5, torch.bfloat16)
        keep = [i for i in range(8) if i != 5]
        assert torch.equal(got[keep], want[keep])


@pytest.mark.parametrize("q_dtype,out_dtype", [(torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32), (torch.float32, torch.float32)])
@pytest.mark.parametrize("d", [128, 192])
def test_attention_cached_tokens_that_only_earlier_rows_see(q_dtype, out_dtype, d):
    """A chain under a window: the first token in reach is seen by node 0 alone.  Whatever its scales are, the other rows stay within their bound."""
    c = dc.attention_case(10, [1000], 6, 8, 2, d, kind="chain", window=700, q_dtype=q_dtype)
    slot = dc.physical(c["tables"], 0, [1000 + 1 - 700], c["page"])
    want, about = dc.attention(c, d**-0.5)
    bound = dc.attention_bound(c, want, about, out_dtype, out_dtype != torch.bfloat16 or q_dtype == torch.float32)
    for k_bad, v_bad in ((1.0, float("nan")), (1.0, float("inf")), (1.0, -float("inf")), (float("nan"), 1.0), (float("inf"), float("inf"))):
        other = dict(c, k_scales=c["k_scales"].clone(), v_scales=c["v_scales"].clone())
        other["k_scales"][slot] *= k_bad
        other["v_scales"][slot] *= v_bad
        got = run_attention(other, d**-0.5, out_dtype).double().cpu()
        assert ((got - want).abs() <= bound)[1:].all()
        assert not torch.isfinite(got[0]).all()


def test_attention_window_over_positions_far_from_the_slots():
    """Nodes whose positions lie well behind their cache slots, as after tokens were dropped from a cache: positions alone decide which nodes a window holds."""
    for rows in (9, 40):
        c = dc.attention_case(11, [100, 37], rows, 8, 2, 128, window=64)
        c["positions"][0] += 50
        c["positions"][1] += 5000
        check_attention(c, torch.bfloat16)
        check_attention(c, torch.float32)


@pytest.mark.parametrize("q_gain,spread", [(30.0, 0.0), (1e-3, 0.0), (1.0, 24.0), (8.0, 12.0)])
@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float32])
def test_attention_magnitudes(q_gain, spread, out_dtype):
    """Peaked and flat rows; V scales over 24 powers of two."""
    check_attention(dc.attention_case(10, [900], 6, 8, 2, 128, q_gain=q_gain, scale_spread=spread, scales=torch.bfloat16), out_dtype)


def test_attention_queries_of_unequal_magnitude():
    """A pair's query scales by its own power of two: one huge row next to ordinary ones."""
    c = dc.attention_case(11, [200], 6, 8, 2, 128)
    want = run_attention(c, 128**-0.5, torch.bfloat16)
    c["q"][2] *= 1e30
    got = run_attention(c, 128**-0.5, torch.bfloat16)
    keep = [0, 1, 3, 4, 5]
    assert torch.equal(got[keep], want[keep])


def test_attention_plan_does_not_change_what_is_read():
    """Any estimate of the longest sequence, with and without the sum; the bound holds for each."""
    c = dc.attention_case(12, [700, 30, 1], 6, 8, 2, 128)
    for total in (False, True):
        check_attention(c, torch.bfloat16, total=total)
    want, about = dc.attention(c, 128**-0.5)
    bound = dc.attention_bound(c, want, about, torch.bfloat16, False)
    q = dev(c["q"])
    for longest in (0, 100, 700):
        got = ops.gqa_draft_attention(q, dev(c["k"]), dev(c["k_scales"]), dev(c["v"]), dev(c["v_scales"]), dev(c["tables"]), ints(c["lens"]), dev(c["masks"]), 8, 2, 128,
                                      c["page"], 128**-0.5, longest, row_counts=ints(c["counts"]), out_dtype=torch.bfloat16)
        assert ((got.double().cpu() - want).abs() <= bound).all()


def test_attention_runs_repeat_bit_for_bit():
    c = dc.attention_case(13, [3000, 900], 10, 16, 4, 128)
    want = run_attention(c, 128**-0.5, torch.float32)
    for _ in range(3):
        assert torch.equal(run_attention(c, 128**-0.5, torch.float32), want)


def test_attention_far_pages():
    """Offsets past 32 bits in the planes: pages in the last of 5 GiB of codes."""
    d, hkv, page, far = 128, 8, 16, 5 << 30
    pool = far // (hkv * d)
    c = dc.attention_case(14, [60], 5, 16, hkv, d, page=page)
    small = c["k"].shape[0]
    planes = {}
    for name in ("k", "v"):
        planes[name] = torch.empty(pool, hkv * d, dtype=torch.int8, device="cuda")
        planes[name + "_scales"] = torch.empty(pool, hkv * 2, dtype=torch.float16, device="cuda")
        planes[name][pool - small :] = dev(c[name])
        planes[name + "_scales"][pool - small :] = dev(c[name + "_scales"])
    want = run_attention(c, d**-0.5, torch.bfloat16)
    got = ops.gqa_draft_attention(dev(c["q"]), planes["k"], planes["k_scales"], planes["v"], planes["v_scales"], dev(c["tables"]) + (pool - small) // page, ints(c["lens"]),
                                  dev(c["masks"]), 16, hkv, d, page, d**-0.5, 60, row_counts=ints(c["counts"]), out_dtype=torch.bfloat16, total_kv_tokens=60)
    assert (pool - small) % page == 0 and torch.equal(got, want)


# ---- verification --------------------------------------------------------------------------------------------------------


def verify_case(seed, batch, rows, vocab, kind, dtype, with_drafts, hot=6):
    gen = torch.Generator().manual_seed(seed)
    parents = dc.tree(gen, batch, rows, kind)
    target = torch.softmax(torch.randn(batch, rows, vocab, generator=gen) * 2.0, -1).to(dtype)
    drafts = None
    few = min(hot, vocab)
    likely = target.float().topk(few, -1).indices
    tokens = torch.randint(0, vocab, (batch, rows), generator=gen)
    for b in range(batch):
        for i in range(1, rows):
            at = int(parents[b, i]) if 0 <= int(parents[b, i]) < i else 0
            tokens[b, i] = likely[b, at, int(torch.randint(0, few, (1,), generator=gen))]
    if with_drafts:
        noise = torch.randn(batch, rows - 1, vocab, generator=gen) * 0.7
        drafts = torch.softmax(torch.log(target[:, :-1].float().clamp(min=1e-30)) + noise, -1).to(dtype)
    uniforms = torch.rand(batch, rows, generator=gen)
    return tokens.to(torch.int32), target, uniforms, parents if kind != "chain" else None, drafts


def check_verify(tokens, target, uniforms, parents, drafts, counts=None, target_dev=None):
    batch, rows = tokens.shape
    path, accepted, out = ops.draft_verify(dev(tokens), dev(target) if target_dev is None else target_dev, dev(uniforms), parents=dev(parents), draft_probs=dev(drafts),
                                           row_counts=None if counts is None else ints(counts))
    want = dc.verify(tokens, target, uniforms, parents, drafts, counts or [rows] * batch)
    for b, (nodes, words) in enumerate(want):
        assert int(accepted[b]) == len(nodes)
        assert path[b].tolist() == nodes + [-1] * (rows - len(nodes))
        assert out[b].tolist() == words + [-1] * (rows - len(words))
    return want


@pytest.mark.parametrize("kind,with_drafts", [("chain", True), ("chain", False), ("tree", False), ("star", False), ("forest", False)])
@pytest.mark.parametrize("batch,rows,vocab", [(1, 1, 7), (4, 2, 1), (9, 6, 1000), (3, 70, 4097), (2, 256, 130), (5, 12, 33001)])
def test_verify(kind, with_drafts, batch, rows, vocab):
    case = verify_case(rows + vocab, batch, rows, vocab, kind, torch.float32, with_drafts and rows > 1)
    check_verify(*case)
    check_verify(*case, counts=[(rows * (b + 1)) // batch for b in range(batch)])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("kind,with_drafts", [("chain", True), ("tree", False)])
def test_verify_types(dtype, kind, with_drafts):
    check_verify(*verify_case(3, 6, 9, 5001, kind, dtype, with_drafts))


def test_verify_row_strides():
    tokens, target, uniforms, parents, drafts = verify_case(4, 5, 6, 777, "chain", torch.float32, True)
    wide = torch.full((5, 6, 800), float("nan"), device="cuda")
    wide[..., :777] = dev(target)
    check_verify(tokens, target, uniforms, parents, drafts, target_dev=wide[..., :777])


def test_verify_borders():
    """Uniforms of 0 and just below 1; certain drafts; tokens past the vocabulary; duplicated siblings; nothing left; nothing at all."""
    tokens = torch.tensor([[0, 1, 1, 2], [0, 9, -1, 3], [0, 1, 2, 3], [0, 0, 0, 0]], dtype=torch.int32)
    target = torch.zeros(4, 4, 5)
    target[:] = torch.tensor([0.5, 0.25, 0.125, 0.125, 0.0])
    target[2, 0] = torch.tensor([0.0, 0.5, 0.25, 0.25, 0.0])  # all of it on the three drafts
    target[3] = 0.0
    star = torch.tensor([[-1, 0, 0, 0]] * 4, dtype=torch.int32)
    for first in (0.0, 0.3, 1.0 - 2.0**-24):
        for later in (0.0, 0.5, 1.0 - 2.0**-24):
            uniforms = torch.full((4, 4), later)
            uniforms[:, 0] = first
            check_verify(tokens, target, uniforms, star, None)
            check_verify(tokens, target, uniforms, None, None)
            check_verify(tokens, target, uniforms, None, target[:, :3].clone())
            check_verify(tokens, target, uniforms, None, target[:, :3].flip(-1).clone())
    target[0, 0, 3] = float("nan")
    target[1, 0, 1] = float("inf")
    check_verify(tokens, target, torch.full((4, 4), 0.5), star, None)


def test_verify_keeps_the_target_distribution():
    """Drafts drawn from q, accepted or replaced: the first token is distributed as p.  60,000 draws of each of six tokens: five standard deviations."""
    gen = torch.Generator().manual_seed(1)
    n, vocab = 60000, 6
    p, q = torch.softmax(torch.randn(2, vocab, generator=gen), -1)
    drafted = torch.multinomial(q, n, replacement=True, generator=gen)
    tokens = torch.stack([torch.zeros(n, dtype=torch.long), drafted], 1).to(torch.int32)
    for drafts in (q.expand(n, 1, vocab).contiguous(), None):
        _, _, out = ops.draft_verify(dev(tokens), p.expand(n, 2, vocab).contiguous().cuda(), torch.rand(n, 2, generator=gen).cuda(), draft_probs=dev(drafts))
        share = torch.bincount(out[:, 0].cpu().long(), minlength=vocab) / n
        assert ((share - p).abs() < 5.0 * (p * (1 - p) / n).sqrt()).all()


# ---- commit --------------------------------------------------------------------------------------------------------------


def check_commit(seed, lens, rows, paths, row_shapes, page=8, ring=0, offset=0):
    gen = torch.Generator().manual_seed(seed)
    batch = len(lens)
    tables, pool = dc.block_tables(gen, [ring or n + rows for n in lens], page)
    planes = []
    for width, dtype in row_shapes:
        flat = torch.randint(-100, 100, (pool * width + 16,), generator=gen).to(dtype)
        planes.append(flat[offset : offset + pool * width].view(pool, width))
    path = torch.full((batch, rows), -1, dtype=torch.int32)
    taken = []
    for b, nodes in enumerate(paths):
        path[b, : len(nodes)] = torch.tensor(nodes, dtype=torch.int32)
        good = 0
        while good < len(nodes) and nodes[good] < rows and nodes[good] >= 0 and (good == 0 or nodes[good] > nodes[good - 1]):
            good += 1
        taken.append(good)
    on_device = [torch.empty(p.numel() + 16, dtype=p.dtype, device="cuda")[offset : offset + p.numel()].view(p.shape).copy_(p) for p in planes]
    lens_out = ops.commit_rows(on_device, dev(tables), ints(lens), dev(path), ints([len(n) for n in paths]), page, ring_capacity=ring)
    assert lens_out.tolist() == [n + t for n, t in zip(lens, taken)]
    for plane, got in zip(planes, on_device):
        want = plane.clone()
        for b, nodes in enumerate(paths):
            sources = dc.physical(tables, b, [lens[b] + i for i in nodes[: taken[b]]], page, ring)
            goals = dc.physical(tables, b, [lens[b] + i for i in range(taken[b])], page, ring)
            want[goals] = plane[sources]
        assert torch.equal(got.cpu(), want)


WIDTHS = [(1024, torch.int8), (16, torch.float16), (64, torch.bfloat16), (3, torch.int16), (5, torch.int8), (20, torch.float32), (1, torch.int8)]


@pytest.mark.parametrize("offset", [0, 1])
def test_commit(offset):
    paths = [[0], [0, 1, 2, 3], [0, 2, 3, 7], [0, 1, 5, 6, 7, 8, 9, 10, 11, 12, 13, 19], [], list(range(20)), [3, 4, 19]]
    check_commit(1, [0, 5, 100, 33, 7, 64, 2], 20, paths, WIDTHS, offset=offset)


def test_commit_ends_at_an_entry_that_is_out_of_order():
    check_commit(2, [10, 20, 3], 9, [[0, 4, 4, 5], [0, 3, 2, 8], [0, 2, 9, 3]], WIDTHS)


def test_commit_ends_behind_the_pages():
    """Tables of two pages for 16 tokens: sequence 0 has room for 11 nodes, sequence 1 for none, sequence 2 for one."""
    gen = torch.Generator().manual_seed(5)
    lens, page, rows = [5, 16, 15], 8, 20
    tables, pool = dc.block_tables(gen, [16, 16, 16], page)
    plane = torch.randint(-100, 100, (pool, 32), generator=gen, dtype=torch.int8)
    path = torch.full((3, rows), -1, dtype=torch.int32)
    path[0, :5] = torch.tensor([0, 3, 10, 11, 15])
    path[1, :3] = torch.tensor([0, 1, 2])
    path[2, :3] = torch.tensor([0, 1, 2])
    got = dev(plane)
    lens_out = ops.commit_rows([got], dev(tables), ints(lens), dev(path), ints([5, 3, 3]), page)
    assert lens_out.tolist() == [8, 16, 16]
    want = plane.clone()
    want[dc.physical(tables, 0, [6, 7], page)] = plane[dc.physical(tables, 0, [8, 15], page)]
    assert torch.equal(got.cpu(), want)


def test_planes_are_different_ones():
    plane = torch.zeros(16, 4, device="cuda")
    with pytest.raises(ValueError, match="twice"):
        ops.commit_planes([plane, plane])
    with pytest.raises(ValueError, match="device"):
        ops.commit_planes([plane, plane.cpu()])


def test_commit_ring_and_many_planes():
    check_commit(3, [10, 95], 6, [[0, 2, 5], [0, 1, 4]], [(32, torch.int8)] * 131 + [(2, torch.int8)] * 5, ring=24)
    check_commit(4, [300], 256, [list(range(0, 256, 2))], [(16, torch.float16)], page=1)


# ---- together ------------------------------------------------------------------------------------------------------------


class Speculation:
    """Two layers of a small model over one batch: drafted nodes go through layout, prologue, attention, verification and commit."""

    hq, hkv, d, page, rows, vocab = 8, 2, 128, 16, 6, 50

    def __init__(self, seed, lens, pages=8):
        gen = torch.Generator().manual_seed(seed)
        self.batch = len(lens)
        self.embed = torch.randn(self.vocab, 2, (self.hq + 2 * self.hkv) * self.d, generator=gen).cuda().bfloat16()
        self.head = (torch.randn(self.hq * self.d, self.vocab, generator=gen) * 0.3).cuda()
        angle = torch.arange(256, dtype=torch.float64)[:, None] / 10000.0 ** (torch.arange(self.d // 2, dtype=torch.float64) * 2 / self.d)
        self.cos, self.sin = angle.cos().float().cuda(), angle.sin().float().cuda()
        self.norm = (torch.randn(self.d, generator=gen) * 0.1).cuda()
        pool = self.batch * pages * self.page
        self.tables = torch.randperm(self.batch * pages, generator=gen).to(torch.int32).view(self.batch, pages).cuda()
        self.planes = []
        for _ in range(2):
            for _ in range(2):
                self.planes += [torch.zeros(pool, self.hkv * self.d, dtype=torch.int8, device="cuda"), torch.zeros(pool, self.hkv * 2, dtype=torch.float16, device="cuda")]
        self.plane_list = ops.commit_planes(self.planes)
        self.lens = ints(lens)
        for b, n in enumerate(lens):  # a prompt
            for layer in range(2):
                x = torch.randn(n, (self.hq + 2 * self.hkv) * self.d, generator=gen).cuda().bfloat16()
                q, k, v = x.split([self.hq * self.d, self.hkv * self.d, self.hkv * self.d], -1)
                if n:
                    ops.gqa_prologue(q.contiguous(), k.contiguous(), v.contiguous(), self.norm, self.norm, self.cos, self.sin, *self.planes[4 * layer : 4 * layer + 4],
                                     self.tables[b], 0, self.hq, self.hkv, self.d, self.d, self.page, q_out_dtype=torch.bfloat16)
        self.positions = None

    def qkv(self, tokens, layer):
        x = self.embed[tokens.flatten().long(), layer]
        return [t.contiguous() for t in x.split([self.hq * self.d, self.hkv * self.d, self.hkv * self.d], -1)]

    def nodes(self, tokens, parents):
        """Target distributions behind every node [batch, rows, vocab]."""
        masks, positions = ops.draft_layout(parents, self.lens)
        total = 0.0
        for layer in range(2):
            cache = self.planes[4 * layer : 4 * layer + 4]
            q, k, v = self.qkv(tokens, layer)
            q = ops.gqa_draft_prologue(q, k, v, self.norm, self.norm, self.cos, self.sin, *cache, self.tables, self.lens, self.hq, self.hkv, self.d, self.d, self.page,
                                       positions=positions, q_out_dtype=torch.bfloat16)
            total = total + ops.gqa_draft_attention(q, *cache, self.tables, self.lens, masks, self.hq, self.hkv, self.d, self.page, self.d**-0.5, 100, out_dtype=torch.float32)
        return torch.softmax(total @ self.head, -1).view(self.batch, -1, self.vocab)

    def step(self, tokens, parents, uniforms):
        probs = self.nodes(tokens, parents)
        path, accepted, out = ops.draft_verify(tokens, probs, uniforms, parents=parents)
        lens = ops.commit_rows(self.plane_list, self.tables, self.lens, path, accepted, self.page)
        self.lens.copy_(lens)
        return probs, path, accepted, out

    def token(self, b, word):
        """One token of one sequence by the operators that exist for single rows: its distribution."""
        n = int(self.lens[b])
        total = 0.0
        for layer in range(2):
            cache = self.planes[4 * layer : 4 * layer + 4]
            q, k, v = self.qkv(torch.tensor([word], device="cuda"), layer)
            q = ops.gqa_prologue(q, k, v, self.norm, self.norm, self.cos, self.sin, *cache, self.tables[b], n, self.hq, self.hkv, self.d, self.d, self.page,
                                 q_out_dtype=torch.bfloat16)
            total = total + ops.gqa_decode(q, *cache, self.tables[b : b + 1], ints([n + 1]), self.hq, self.hkv, self.d, self.page, self.d**-0.5, n + 1)
        self.lens[b] += 1
        return torch.softmax(total @ self.head, -1)[0]


def test_steps_agree_with_one_token_at_a_time():
    """Drafted and verified steps leave the cache and the distributions that single-token decoding of the accepted tokens leaves: the same bits in the
    pages, and distributions whose logits come from two f32 attentions, each within its bound of the other's."""
    lens = [0, 19, 45]
    fast, slow = Speculation(1, lens), Speculation(1, lens)
    gen = torch.Generator().manual_seed(2)
    last = [3, 7, 11]
    done = [[] for _ in lens]
    for step in range(4):
        parents = dc.tree(gen, 3, fast.rows, "tree")
        tokens = torch.randint(0, fast.vocab, (3, fast.rows), generator=gen, dtype=torch.int64)
        tokens[:, 0] = torch.tensor(last)
        uniforms = torch.rand(3, fast.rows, generator=gen)
        uniforms[:, 1:] *= 0.05  # accept often
        before = fast.lens.tolist()
        probs, path, accepted, out = fast.step(dev(tokens.to(torch.int32)), dev(parents), dev(uniforms))
        assert fast.lens.tolist() == [n + int(a) for n, a in zip(before, accepted)]
        for b in range(3):
            for i in range(int(accepted[b])):
                node = int(path[b, i])
                want = slow.token(b, int(tokens[b, node]))
                assert torch.allclose(probs[b, node], want, rtol=1e-3, atol=1e-6)
            done[b].append(int(accepted[b]))
            last[b] = int(out[b, int(accepted[b]) - 1])
    assert slow.lens.tolist() == fast.lens.tolist() and max(max(d) for d in done) > 1
    for b in range(3):
        at = dc.physical(fast.tables.cpu(), b, range(int(fast.lens[b])), fast.page).cuda()
        for one, other in zip(fast.planes, slow.planes):
            assert torch.equal(one[at], other[at])


def test_a_recorded_step_replays_with_other_trees_and_lengths():
    """One graph of a whole step; trees, tokens and lengths change between its replays, eager work runs between them, and every replay has the eager
    run's bits."""
    lens = [5, 30]
    captured, eager = Speculation(3, lens), Speculation(3, lens)
    gen = torch.Generator().manual_seed(4)
    tokens, parents = torch.zeros(2, 6, dtype=torch.int32, device="cuda"), dev(dc.tree(gen, 2, 6, "chain"))
    uniforms = torch.zeros(2, 6, device="cuda")
    keep = [t.clone() for t in captured.planes] + [captured.lens.clone()]
    captured.step(tokens, parents, uniforms)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        result = captured.step(tokens, parents, uniforms)
    for t, was in zip(captured.planes + [captured.lens], keep):
        t.copy_(was)
    for kind in ("tree", "star", "chain", "tree", "forest"):
        parents.copy_(dc.tree(gen, 2, 6, kind))
        tokens.copy_(torch.randint(0, 50, (2, 6), generator=gen))
        uniforms.copy_(torch.rand(2, 6, generator=gen) * 0.2)
        graph.replay()
        want = eager.step(tokens, parents, uniforms)
        torch.cuda.synchronize()
        for got, right in zip(result, want):
            assert torch.equal(got, right)
        assert torch.equal(captured.lens, eager.lens)
        for one, other in zip(captured.planes, eager.planes):
            assert torch.equal(one, other)


def test_two_streams_at_once():
    """Calls on two streams share nothing: each with its own workspace gets the bits it gets alone."""
    cases = [dc.attention_case(20 + i, [1500, 300], 8, 16, 4, 128) for i in range(2)]
    verifies = [verify_case(30 + i, 6, 8, 9001, "tree", torch.float32, False) for i in range(2)]
    want = [run_attention(c, 128**-0.5, torch.bfloat16) for c in cases]
    want_verify = [ops.draft_verify(dev(v[0]), dev(v[1]), dev(v[2]), parents=dev(v[3])) for v in verifies]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got, got_verify = [[], []], [[], []]
    for _ in range(3):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[i].append(run_attention(cases[i], 128**-0.5, torch.bfloat16))
                v = verifies[i]
                got_verify[i].append(ops.draft_verify(dev(v[0]), dev(v[1]), dev(v[2]), parents=dev(v[3])))
    torch.cuda.synchronize()
    for i in range(2):
        for out in got[i]:
            assert torch.equal(out, want[i])
        for out in got_verify[i]:
            assert all(torch.equal(a, b) for a, b in zip(out, want_verify[i]))


def test_prologue_default_rows_are_those_of_a_tensor_program():
    """The entry point's own quantizer: the bits that the formula has where a tensor program on this device evaluates it, with bf16 and f16 values whose groups
    have ordinary maxima (half a maximum lies on a tie of two codes).  METAL_GQA at the same values has the bits of the prologue and the append of single
    sequences, and so has RECIPROCAL_GQA, which those take as well."""
    gen = torch.Generator().manual_seed(77)
    batch, rows, heads, d, page = 24, 48, 8, 128, 16
    nodes, cols = batch * rows, heads * d
    tables = torch.randperm(batch * 3, generator=gen).to(torch.int32).view(batch, 3)
    slots = (tables.long()[..., None] * page + torch.arange(page)).view(batch * rows).cuda()
    norm = (torch.randn(d, generator=gen) * 0.1).cuda()
    for src in (torch.bfloat16, torch.float16, torch.float32):
        q, k, v = torch.randn(3, nodes, cols, generator=gen).to(src).cuda()
        empty = lambda: [torch.zeros(nodes, cols, dtype=torch.int8, device="cuda"), torch.zeros(nodes, cols // 64, dtype=torch.float16, device="cuda")]

        def drafted(**rule):
            planes = empty() + empty()
            out = ops.gqa_draft_prologue(q, k, v, norm, norm, None, None, *planes, dev(tables), ints([0] * batch), heads, heads, d, 0, page, **rule)
            return out, [p[slots] for p in planes]

        out, (k_codes, k_scales, v_codes, v_scales) = drafted()
        groups = v.float().view(nodes, -1, 64)
        most = groups.abs().amax(-1)
        step = most / 127.0
        assert torch.equal(step, most * torch.tensor(1.0 / 127.0, device="cuda"))
        assert torch.equal(v_scales, step.half())
        assert torch.equal(v_codes.view(groups.shape), torch.round(groups * (1.0 / step)[..., None]).clamp(-127, 127).to(torch.int8))
        results = {}
        for rule in (capi.QUANT_METAL_GQA, capi.QUANT_RECIPROCAL_GQA):
            results[rule] = drafted(rule=rule)
            single = empty() + empty()
            single_out = ops.gqa_prologue(q, k, v, norm, norm, None, None, *single, None, 0, heads, heads, d, 0, page, rule=rule)
            assert torch.equal(single_out, results[rule][0])
            for one, other in zip(single, results[rule][1]):
                assert torch.equal(one, other)
            appended = empty()
            ops.q8g64_append(v, *appended, None, 0, page, rule)
            assert torch.equal(appended[0], single[2]) and torch.equal(appended[1], single[3])
        for one, other in zip([out, k_codes, k_scales, v_codes, v_scales], [results[capi.QUANT_RECIPROCAL_GQA][0], *results[capi.QUANT_RECIPROCAL_GQA][1]]):
            assert torch.equal(one, other)
        if src == torch.bfloat16:  # the two rules do differ here
            assert not torch.equal(results[capi.QUANT_METAL_GQA][1][2], v_codes)


@pytest.mark.parametrize("shift", [0, 1])
def test_prologue_lengths_at_the_end_of_their_range(shift):
    """Nodes of a sequence whose length is no length (-1): none of them has a place in the sequence's pages, the first pages among them."""
    gen = torch.Generator().manual_seed(5)
    q, k, v = (torch.randn(8, 64, generator=gen).cuda() for _ in range(3))
    codes = [torch.zeros(24 * 64 + 16, dtype=torch.int8, device="cuda")[shift : 24 * 64 + shift].view(24, 64) for _ in range(2)]
    steps = [torch.zeros(24, 1, dtype=torch.float16, device="cuda") for _ in range(2)]
    tables = torch.tensor([[0, 1, 2], [5, 4, 3]], dtype=torch.int32)
    ops.gqa_draft_prologue(q, k, v, None, None, None, None, codes[0], steps[0], codes[1], steps[1], dev(tables), ints([-1, 2]), 1, 1, 64, 0, 4)
    written = torch.zeros(24, dtype=torch.bool)
    written[dc.physical(tables, 1, range(2, 6), 4)] = True
    for plane in codes + steps:
        assert torch.equal((plane != 0).any(-1).cpu(), written)
