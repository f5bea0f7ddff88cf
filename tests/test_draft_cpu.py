"""Refusals and plans of the drafted-token entry points: every bad call ends on the host, before anything is launched (no GPU here)."""
import ctypes as C

import pytest
import torch

from tests import draft_cases as dc
from zllm_amd import capi

FAKE = 0x1000  # an address that is never read


def refused(rc, *words):
    assert rc < 0
    text = capi.last_error()
    assert all(w in text for w in words), text


def fill(kind, **more):
    args = kind()
    for name, ctype in kind._fields_:
        if ctype is capi._ptr:
            setattr(args, name, FAKE)
    for name, value in more.items():
        setattr(args, name, value)
    return args


def attention_args(**more):
    kw = dict(batch=2, rows=5, num_heads=8, num_kv_heads=2, head_dim=128, table_stride=10, max_kv_len=100, block_tokens=16, score_scale=0.1, softcap=0.0,
              kv_format=capi.KV_Q8G64, scale_dtype=capi.SCALE_F16, q_dtype=capi.DTYPE_BF16, out_dtype=capi.DTYPE_BF16, gate=None)
    kw.update(more)
    return fill(capi.GqaDraftAttentionArgs, **kw)


def test_layout_refusals():
    lib = capi.load()
    good = dict(batch=2, rows=5)
    refused(lib.zllm_attn_draft_layout(None, None), "null")
    for name in ("parents", "kv_lens", "masks", "positions"):
        refused(lib.zllm_attn_draft_layout(C.byref(fill(capi.DraftLayoutArgs, **good, **{name: None})), None), "null")
    for bad in (dict(batch=0), dict(rows=0), dict(rows=257)):
        refused(lib.zllm_attn_draft_layout(C.byref(fill(capi.DraftLayoutArgs, **{**good, **bad})), None), "shape")
    refused(lib.zllm_attn_draft_layout(C.byref(fill(capi.DraftLayoutArgs, **good, masks=FAKE + 4)), None), "aligned")


def test_prologue_refusals():
    lib = capi.load()
    good = dict(batch=2, rows=5, num_heads=8, num_kv_heads=2, head_dim=128, rotary_dim=128, rope_table_rows=64, table_stride=4, block_tokens=16, eps=1e-6,
                src_dtype=capi.DTYPE_BF16, q_out_dtype=capi.DTYPE_BF16)
    call = lambda **bad: lib.zllm_attn_gqa_draft_prologue(C.byref(fill(capi.GqaDraftPrologueArgs, **{**good, **bad})), None)
    refused(lib.zllm_attn_gqa_draft_prologue(None, None), "null")
    for name in ("q", "k", "v", "q_out", "k_plane", "v_plane", "k_scales", "v_scales", "tables", "kv_lens"):
        refused(call(**{name: None}), "null")
    for bad in (dict(batch=0), dict(rows=0), dict(rows=257), dict(num_heads=0), dict(num_kv_heads=0), dict(head_dim=96), dict(head_dim=320), dict(block_tokens=0),
                dict(table_stride=0), dict(batch=1 << 25, rows=256)):
        refused(call(**bad), "shape")
    for bad in (dict(rotary_dim=7), dict(rotary_dim=130), dict(cosine=None), dict(sine=None), dict(rope_table_rows=0)):
        refused(call(**bad), "rotary")
    refused(call(eps=0.0), "eps")
    for bad in (dict(ring_capacity=4), dict(ring_capacity=65)):
        refused(call(**bad), "ring")
    refused(call(kv_format=2), "kv_format")
    for bad in (dict(rule=4), dict(rule=-1), dict(src_dtype=3), dict(q_out_dtype=-1)):
        refused(call(**bad), "unknown")


def test_attention_refusals():
    lib = capi.load()
    size = lambda **bad: lib.zllm_attn_gqa_draft_attention_workspace_bytes(C.byref(attention_args(**bad)))
    call = lambda **bad: lib.zllm_attn_gqa_draft_attention(C.byref(attention_args(workspace_bytes=1 << 40, **bad)), None)
    assert size() > 0
    for bad, word in ((dict(batch=0), "shape"), (dict(rows=0), "shape"), (dict(rows=257), "shape"), (dict(num_heads=0), "shape"), (dict(num_kv_heads=0), "shape"),
                      (dict(num_heads=9), "shape"), (dict(num_heads=514), "shape"), (dict(head_dim=96), "head_dim"), (dict(kv_format=1, head_dim=64), "head_dim"),
                      (dict(kv_format=2), "head_dim"), (dict(scale_dtype=3), "scales"), (dict(block_tokens=0), "non-zero"), (dict(table_stride=0), "non-zero"),
                      (dict(max_kv_len=0x7fffff00, table_stride=1 << 30), "below"), (dict(max_kv_len=156), "cannot cover"),
                      (dict(ring_capacity=64), "ring"), (dict(ring_capacity=20, window=17), "ring"), (dict(ring_capacity=200, window=17), "ring"),
                      (dict(window=0x7fffff01), "window"), (dict(score_scale=0.0), "score_scale"), (dict(score_scale=float("nan")), "score_scale"),
                      (dict(softcap=-1.0), "softcap"), (dict(softcap=float("inf")), "softcap"), (dict(q_dtype=3), "q_dtype"), (dict(out_dtype=-1), "out_dtype")):
        assert size(**bad) == 0
        refused(call(**bad), word)
    for name in ("q", "k_plane", "v_plane", "k_scales", "v_scales", "tables", "kv_lens", "out", "workspace"):
        refused(call(**{name: None}), "null")
    refused(call(window=9, positions=None), "null")
    for name in ("q", "k_plane", "v_plane", "out", "workspace"):
        refused(call(**{name: FAKE + 8}), "aligned")
    refused(call(masks=FAKE + 4), "aligned")
    refused(call(k_scales=FAKE + 2), "aligned")
    refused(call(gate=FAKE, gate_cols=3), "gate")
    refused(call(gate=FAKE, gate_cols=1, gate_dtype=capi.DTYPE_F16), "gate")
    need = size()
    refused(lib.zllm_attn_gqa_draft_attention(C.byref(attention_args(workspace_bytes=need - 1)), None), "workspace")
    refused(call(batch=1 << 26, rows=256, table_stride=100), "too many")


def test_attention_workspace_follows_the_tokens_there_are():
    """One long sequence among short ones: with the sum of their lengths the records are for the parts there are."""
    lib = capi.load()
    kw = dict(batch=24, rows=8, max_kv_len=150000, table_stride=150000 // 16 + 1)
    without = lib.zllm_attn_gqa_draft_attention_workspace_bytes(C.byref(attention_args(**kw)))
    with_sum = lib.zllm_attn_gqa_draft_attention_workspace_bytes(C.byref(attention_args(**kw, total_kv_tokens=160000)))
    assert with_sum < without


def test_verify_refusals():
    lib = capi.load()
    good = dict(batch=2, rows=5, vocab=100, parents=None)
    size = lambda **bad: lib.zllm_attn_draft_verify_workspace_bytes(C.byref(fill(capi.DraftVerifyArgs, **{**good, **bad})))
    call = lambda **bad: lib.zllm_attn_draft_verify(C.byref(fill(capi.DraftVerifyArgs, workspace_bytes=1 << 40, **{**good, **bad})), None)
    assert size() > 0
    for bad, word in ((dict(batch=0), "shape"), (dict(batch=65536), "shape"), (dict(rows=0), "shape"), (dict(rows=257), "shape"), (dict(vocab=0), "shape"),
                      (dict(vocab=1 << 31), "shape"), (dict(target_dtype=3), "dtype"), (dict(draft_dtype=-1), "dtype"), (dict(parents=FAKE), "chain"),
                      (dict(target_stride=99), "shorter"), (dict(draft_stride=99), "shorter")):
        assert size(**bad) == 0
        refused(call(**bad), word)
    refused(lib.zllm_attn_draft_verify(None, None), "null")
    for name in ("tokens", "target_probs", "uniforms", "path", "accepted", "out_tokens", "workspace"):
        refused(call(**{name: None}), "null")
    refused(call(workspace=FAKE + 8), "workspace")
    refused(lib.zllm_attn_draft_verify(C.byref(fill(capi.DraftVerifyArgs, workspace_bytes=size() - 1, **good)), None), "workspace")


def test_commit_refusals():
    lib = capi.load()

    def call(planes=((FAKE, 64),), **bad):
        array = (capi.KvPlane * max(1, len(planes)))(*[capi.KvPlane(*p) for p in planes])
        kw = dict(plane_count=len(planes), batch=2, rows=5, table_stride=4, block_tokens=16, new_lens=FAKE + 64)
        kw.update(bad)
        args = fill(capi.CommitRowsArgs, **kw)
        if "planes_pointer" not in bad:
            args.planes = array
        return lib.zllm_attn_commit_rows(C.byref(args), None)

    refused(lib.zllm_attn_commit_rows(None, None), "null")
    for name in ("tables", "kv_lens", "path", "accepted"):
        refused(call(**{name: None}), "null")
    for bad in (dict(planes=()), dict(batch=0), dict(rows=0), dict(rows=257), dict(table_stride=0), dict(block_tokens=0)):
        refused(call(**bad), "shape")
    refused(call(new_lens=FAKE), "kv_lens")
    refused(call(new_lens=FAKE + 128, accepted=FAKE + 128), "accepted")
    for bad in (dict(ring_capacity=4), dict(ring_capacity=40, table_stride=2)):
        refused(call(**{"rows": 6, "block_tokens": 16, **bad}), "ring")
    for planes in (((None, 64),), ((FAKE, 64), (FAKE, 0)), ((FAKE, 1 << 31),)):
        refused(call(planes=planes), "plane")


def test_python_entry_points_check_their_tensors():
    from zllm_amd import ops

    host = torch.zeros(2, 3, dtype=torch.int32)
    with pytest.raises(ValueError, match="parents"):
        ops.draft_layout(host, host[:, 0])
    with pytest.raises(ValueError, match="target_probs"):
        ops.draft_verify(host, torch.zeros(2, 3, 7), torch.zeros(2, 3))
    with pytest.raises(ValueError, match="plane"):
        ops.commit_planes([torch.zeros(4, 4)])
    with pytest.raises(ValueError, match="rows"):
        ops.gqa_draft_attention(torch.zeros(5, 128), None, None, None, None, host, host[:, 0], None, 1, 1, 128, 16, 1.0, 10)


def test_definitions_of_the_cases():
    """The 64-bit walk on small vectors by hand."""
    tokens = torch.tensor([[5, 1, 2, 3]], dtype=torch.int32)
    target = torch.tensor([[[0.1, 0.6, 0.2, 0.1]] * 4])
    # node 1 rejected (0.9 >= 0.6), then node 2: 0.4 * 0.4 < 0.2 passes; node 3 hangs on node 1: never reached; next token by 0.75 of row 2
    parents = torch.tensor([[-1, 0, 0, 1]], dtype=torch.int32)
    uniforms = torch.tensor([[0.75, 0.9, 0.4, 0.0]])
    assert dc.verify(tokens, target, uniforms, parents, None, [4]) == [([0, 2], [2, 2])]
    # a chain drawn from q: 0.9 * 0.5 < 0.6 passes, then 0.5 * 0.9 >= 0.2 ends it; of max(p - q, 0) = (0.05, 0.55, 0, 0.1): 0.75 of 0.7 lies in token 1
    q = torch.tensor([[[0.2, 0.5, 0.2, 0.1], [0.05, 0.05, 0.9, 0.0], [0.25, 0.25, 0.25, 0.25]]])
    assert dc.verify(tokens, target, torch.tensor([[0.75, 0.9, 0.5, 0.0]]), None, q, [4]) == [([0, 1], [1, 1])]
    sees, depth = dc.ancestors(torch.tensor([[-1, 0, 1, 0, 3]], dtype=torch.int32), [5])
    assert dc.pack(sees).flatten().tolist() == [1, 3, 7, 9, 25] and depth.flatten().tolist() == [0, 1, 2, 1, 2]


def test_distributions_whose_rows_overlap_are_refused():
    """Rows of stride 0 (one distribution expanded over the nodes) or shorter than the vocabulary: the kernel takes 0 for the vocabulary and would read past them."""
    from zllm_amd import ops

    vocab = 7
    one = torch.rand(vocab)
    for t in (one.expand(4, 3, vocab), torch.rand(4, 1, vocab).expand(4, 3, vocab), torch.rand(1, 3, vocab).expand(4, 3, vocab), torch.rand(20).as_strided((4, 3, vocab), (3, 1, 1)),
              torch.rand(1, 1).expand(4, 3, 1), torch.rand(4, 3, 2 * vocab)[..., ::2]):
        with pytest.raises(ValueError, match="probs"):
            ops._prob_rows(t, "target_probs", 12, t.shape[-1], -1)
    assert ops._prob_rows(torch.rand(4, 3, vocab), "p", 12, vocab, -1) == vocab
    assert ops._prob_rows(torch.rand(4, 3, 9)[..., :vocab], "p", 12, vocab, -1) == 9
    assert ops._prob_rows(one.expand(1, 1, vocab), "p", 1, vocab, -1) == vocab
    assert ops._prob_rows(torch.rand(12, vocab)[::2].view(2, 3, vocab), "p", 6, vocab, -1) == 2 * vocab
    assert ops._prob_rows(torch.rand(4, 3, 1), "p", 12, 1, -1) == 1


def test_planes_of_other_types_or_widths_are_refused():
    """A cache's planes against the call's formats: what does not fit would be read or written past its end, or as other values."""
    from zllm_amd import ops

    codes, f16_scales = torch.zeros(32, 256, dtype=torch.int8), torch.zeros(32, 4, dtype=torch.float16)
    good = dict(k_plane=codes, k_scales=f16_scales, v_plane=codes, v_scales=f16_scales, num_kv_heads=2, head_dim=128, kv_format=capi.KV_Q8G64, scales=torch.float16, device=-1)
    check = lambda **bad: ops._cache_planes(**{**good, **bad})
    assert check() == tuple(t.data_ptr() for t in (codes, f16_scales, codes, f16_scales))
    assert check(k_plane=codes.view(2, 16, 2, 128), k_scales=f16_scales.view(2, 16, 4))[0] == codes.data_ptr()  # any shape of whole rows
    assert check(k_plane=None)[0] is None  # the C call names null pointers
    for name, bad in (("k_scales", f16_scales.bfloat16()), ("v_scales", f16_scales.float()), ("k_plane", codes.half()), ("v_plane", codes.float()),
                      ("k_plane", torch.zeros(32, 250, dtype=torch.int8)), ("v_plane", codes[:16]), ("k_scales", f16_scales[:, :2].contiguous()), ("v_scales", f16_scales[:31]),
                      ("k_plane", codes[:, ::2]), ("k_plane", codes[:0])):
        with pytest.raises(ValueError, match=name[2:]):
            check(**{name: bad})
    for scales in (torch.bfloat16, torch.float32):
        with pytest.raises(ValueError, match="scales"):
            check(scales=scales)
    with pytest.raises(ValueError, match="plane"):
        check(head_dim=192)
    halves = torch.zeros(32, 256, dtype=torch.float16)
    f16 = dict(k_plane=halves, k_scales=None, v_plane=halves, v_scales=None, kv_format=capi.KV_F16)
    assert check(**f16) == (halves.data_ptr(), None, halves.data_ptr(), None)
    for bad in (halves.bfloat16(), codes, halves.float()):
        with pytest.raises(ValueError, match="plane"):
            check(**{**f16, "v_plane": bad})
    assert [ops._RULE_SCALES[rule] for rule in range(4)] == [torch.bfloat16, torch.float16, torch.float32, torch.float16]


def test_commit_planes_are_rows():
    """[layers, rows, columns] is no plane: its first dimension would be taken for tokens."""
    from zllm_amd import ops

    for plane in (torch.zeros(2, 8, 4), torch.zeros(8), torch.zeros(8, 4)[:, ::2]):
        with pytest.raises(ValueError, match="plane"):
            ops._commit_plane(plane, -1)
    assert ops._commit_plane(torch.zeros(8, 4, dtype=torch.float16), -1) == 8


def test_batches_of_no_sequences():
    from zllm_amd import ops

    none, tables = torch.zeros(0, dtype=torch.int32), torch.zeros(0, 4, dtype=torch.int32)
    with pytest.raises(ValueError, match="rows"):
        ops.gqa_draft_attention(torch.zeros(5, 128), None, None, None, None, tables, none, None, 1, 1, 128, 16, 1.0, 10)
    with pytest.raises(ValueError, match="rows"):
        ops.gqa_draft_prologue(torch.zeros(5, 128), None, None, None, None, None, None, None, None, None, None, tables, none, 1, 1, 128, 0, 16)


def test_calls_larger_than_a_grid_are_refused():
    """A grid has fewer than 2^32 threads: sizes just above, for each kernel of a call, end as a refusal that names them before anything is launched."""
    lib = capi.load()
    refused(lib.zllm_attn_draft_layout(C.byref(fill(capi.DraftLayoutArgs, batch=1 << 24, rows=256)), None), "too many")
    refused(lib.zllm_attn_draft_layout(C.byref(fill(capi.DraftLayoutArgs, batch=1 << 26, rows=64)), None), "too many")
    good = dict(rows=256, num_heads=2, num_kv_heads=1, head_dim=192, rotary_dim=0, table_stride=4, block_tokens=16, eps=1e-6)
    prologue = lambda **more: lib.zllm_attn_gqa_draft_prologue(C.byref(fill(capi.GqaDraftPrologueArgs, **{**good, **more})), None)
    refused(prologue(batch=1 << 16), "too many")
    refused(prologue(batch=1 << 16, head_dim=128, k=FAKE + 2), "too many")  # values that are not 16-byte aligned
    refused(prologue(batch=1 << 19, head_dim=128), "too many")
    call = lambda **more: lib.zllm_attn_gqa_draft_attention(C.byref(attention_args(workspace_bytes=1 << 40, **more)), None)
    refused(call(batch=1 << 21, rows=1, num_heads=8, num_kv_heads=8), "too many")
    refused(call(batch=1 << 18, rows=256, num_heads=1, num_kv_heads=1, head_dim=256, max_kv_len=0, table_stride=16), "too many")  # the merge
