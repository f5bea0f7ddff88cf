"""Torch-tensor plumbing over the C ABI (device memory + the current HIP stream only).

Every function builds the argument block of include/zllm_attn.h from tensors and calls
the library; no arithmetic happens here.
"""
from __future__ import annotations

import ctypes as C

import torch

from . import capi

_DTYPE = {torch.float32: capi.DTYPE_F32, torch.bfloat16: capi.DTYPE_BF16, torch.float16: capi.DTYPE_F16}


# A decode step of a short context is a few launches of a few microseconds: what a call costs here counts as much as its
# kernels.  Argument blocks are filled by one constructor call, in the order of their fields, with plain integers for pointers.
def _ptr(t):
    return None if t is None else t.data_ptr()


# torch.cuda.current_stream() without the Stream object: 0.3 us a call instead of 2.7.  Not a public name: a torch without it takes the public way
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _stream():
    return torch.cuda.current_stream().cuda_stream if _raw_stream is None else _raw_stream(torch.cuda.current_device())


def _dev(t, name):
    if t is not None and (not t.is_cuda or not t.is_contiguous()):
        raise ValueError(f"{name} must be a contiguous device tensor")
    return t


def _workspace(preferred, least_of, args, device):
    """Device memory of the size with which a call is fastest, or of the least with which it runs where the device has not that much left."""
    try:
        return torch.empty(preferred, dtype=torch.uint8, device=device)
    except torch.OutOfMemoryError:
        least = least_of(C.byref(args))
        if least >= preferred:
            raise
    return torch.empty(max(least, 256), dtype=torch.uint8, device=device)


def init(device: int = 0) -> int:
    cu = C.c_int(0)
    capi.check(capi.load().zllm_attn_init(device, C.byref(cu)))
    return cu.value


def q8g64_append(src, codes, scales, table, position, block_tokens, rule, ring_capacity=0, positions=None):
    """Quantize rows of `src` [T, cols] into the paged planes (zllm_attn_q8g64_append)."""
    _dev(src, "src"), _dev(codes, "codes"), _dev(scales, "scales"), _dev(table, "table")
    args = capi.Q8AppendArgs(_ptr(src), _ptr(codes), _ptr(scales), _ptr(table), _ptr(positions), position,
                             src.shape[0], src.shape[1], block_tokens, ring_capacity, _DTYPE[src.dtype], rule)
    capi.check(capi.load().zllm_attn_q8g64_append(C.byref(args), _stream()))


def gqa_prologue(q, k, v, q_norm, k_norm, cos, sin, k_codes, k_scales, v_codes, v_scales, table, position, num_heads,
                 num_kv_heads, head_dim, rotary_dim, block_tokens, eps=1e-6, weight_offset=1.0, rule=capi.QUANT_METAL_GQA,
                 split_half=True, q_out_dtype=torch.float32, ring_capacity=0, positions=None):
    """Per-head RMSNorm + RoPE of Q and K, Q out as a tensor, K and V quantized into the pages (zllm_attn_gqa_prologue)."""
    rows = q.shape[0]
    q_out = q.new_empty((rows, num_heads * head_dim), dtype=q_out_dtype)
    args = capi.GqaPrologueArgs(
        q.data_ptr(), _ptr(k), _ptr(v), _ptr(q_norm), _ptr(k_norm), _ptr(cos), _ptr(sin), q_out.data_ptr(), _ptr(k_codes),
        _ptr(k_scales), _ptr(v_codes), _ptr(v_scales), _ptr(table), _ptr(positions), rows, num_heads, num_kv_heads, head_dim, rotary_dim,
        0 if cos is None else cos.shape[0], position, block_tokens, ring_capacity, eps, weight_offset, _DTYPE[q.dtype],
        _DTYPE[q_out_dtype], rule, int(split_half))
    capi.check(capi.load().zllm_attn_gqa_prologue(C.byref(args), _stream()))
    return q_out


def half_append(src, cache, table, position, block_tokens, ring_capacity=0):
    _dev(src, "src"), _dev(cache, "cache"), _dev(table, "table")
    dst = capi.DTYPE_BF16 if cache.dtype == torch.bfloat16 else capi.DTYPE_F16
    args = capi.HalfAppendArgs(_ptr(src), _ptr(cache), _ptr(table), position, src.shape[0], src.shape[1],
                               block_tokens, ring_capacity, _DTYPE[src.dtype], dst)
    capi.check(capi.load().zllm_attn_half_append(C.byref(args), _stream()))


def mla_append(latent, k_rope, latent_codes, latent_scales, rope_cache, table, position, block_tokens, cos=None,
               sin=None, rotary_dim=0, rotary_layout=capi.ROTARY_SPLIT_HALF, rope_position=0, positions=None):
    for name, t in (("latent", latent), ("k_rope", k_rope), ("latent_codes", latent_codes),
                    ("latent_scales", latent_scales), ("rope_cache", rope_cache)):
        _dev(t, name)
    args = capi.MlaAppendArgs(_ptr(latent), _ptr(k_rope), _ptr(cos), _ptr(sin), _ptr(latent_codes),
                              _ptr(latent_scales), _ptr(rope_cache), _ptr(table), _ptr(positions), position,
                              rope_position, latent.shape[0], latent.shape[1], k_rope.shape[1], rotary_dim,
                              rotary_layout, block_tokens)
    capi.check(capi.load().zllm_attn_mla_append(C.byref(args), _stream()))


def gather_rows(plane, table, first, count, row_bytes, block_tokens, ring_capacity=0):
    out = torch.empty((count, row_bytes), dtype=torch.uint8, device=plane.device)
    args = capi.GatherArgs(_ptr(plane), _ptr(out), _ptr(table), first, count, row_bytes, block_tokens, ring_capacity)
    capi.check(capi.load().zllm_attn_gather_rows(C.byref(args), _stream()))
    return out


def scatter_rows(plane, rows, table, first, block_tokens, ring_capacity=0):
    """plane[paged_row(first + r)] = rows[r] (zllm_attn_scatter_rows); `rows` is a dense [count, row_bytes] uint8 tensor."""
    args = capi.ScatterArgs(_ptr(plane), _ptr(rows), _ptr(table), first, rows.shape[0], rows.shape[1], block_tokens, ring_capacity)
    capi.check(capi.load().zllm_attn_scatter_rows(C.byref(args), _stream()))


def _gqa_decode_args(launched, q, k_plane, k_scales, v_plane, v_scales, tables, kv_lens, num_heads, num_kv_heads, head_dim,
                     block_tokens, score_scale, max_kv_len, first_visible=None, softcap=0.0, ring_capacity=0,
                     kv_format=capi.KV_Q8G64, scale_dtype=capi.SCALE_F16, out=None, workspace=None, total_kv_tokens=0, gate=None):
    batch = q.shape[0]
    if out is None:
        out = q.new_empty((batch, num_heads * head_dim), dtype=torch.float32)
    args = capi.GqaDecodeArgs(
        q.data_ptr(), _ptr(k_plane), _ptr(k_scales), _ptr(v_plane), _ptr(v_scales), _ptr(tables), _ptr(kv_lens), _ptr(first_visible),
        out.data_ptr(), None, 0, batch, num_heads, num_kv_heads, head_dim, 0 if tables is None else tables.shape[1], max_kv_len,
        total_kv_tokens, block_tokens, ring_capacity, score_scale, softcap, kv_format, scale_dtype, _DTYPE[q.dtype])
    if gate is not None:
        args.gate, args.gate_cols, args.gate_dtype = gate.data_ptr(), gate.shape[1], _DTYPE[gate.dtype]
    if not launched or workspace is None:  # a call that launches with the caller's workspace is checked by the launch itself
        need = capi.load().zllm_attn_gqa_decode_workspace_bytes(C.byref(args))
        if need == 0:
            raise capi.ZllmAttnError(-1, capi.last_error())
    if workspace is False:  # the static-scratch entry point ignores both fields
        return args, out, None
    if workspace is None:
        workspace = torch.empty(need, dtype=torch.uint8, device=q.device)
    args.workspace, args.workspace_bytes = workspace.data_ptr(), workspace.numel()
    return args, out, workspace


def gqa_decode_args(q, k_plane, k_scales, v_plane, v_scales, tables, kv_lens, num_heads, num_kv_heads, head_dim,
                    block_tokens, score_scale, max_kv_len, first_visible=None, softcap=0.0, ring_capacity=0,
                    kv_format=capi.KV_Q8G64, scale_dtype=capi.SCALE_F16, out=None, workspace=None, total_kv_tokens=0, gate=None):
    return _gqa_decode_args(False, q, k_plane, k_scales, v_plane, v_scales, tables, kv_lens, num_heads, num_kv_heads, head_dim,
                            block_tokens, score_scale, max_kv_len, first_visible, softcap, ring_capacity, kv_format, scale_dtype, out,
                            workspace, total_kv_tokens, gate)


def gqa_decode(*a, **kw):
    """Batched GQA decode over the paged cache (zllm_attn_gqa_decode).  Returns f32 [batch, Hq*d]."""
    args, out, workspace = _gqa_decode_args(True, *a, **kw)
    capi.check(capi.load().zllm_attn_gqa_decode(C.byref(args), _stream()))
    return out


def gqa_decode_static(*a, **kw):
    """zllm_attn_gqa_decode_static: the same call over the library's static device array (no workspace of the caller's)."""
    args, out, _ = gqa_decode_args(*a, workspace=False, **kw)
    capi.check(capi.load().zllm_attn_gqa_decode_static(C.byref(args), _stream()))
    return out


def gqa_prefill_chunk_args(q, k_plane, k_scales, v_plane, v_scales, table, position, num_heads, num_kv_heads, head_dim,
                           block_tokens, score_scale, window=0, softcap=0.0, kv_format=capi.KV_Q8G64,
                           scale_dtype=capi.SCALE_F16, out_dtype=torch.float32, gate=None, visible_ends=None, workspace=True,
                           visible_starts=None):
    """The argument block of zllm_attn_gqa_prefill_chunk, the output tensor and the workspace tensor (None without one):
    for callers that launch the same call many times."""
    rows = q.shape[0]
    out = q.new_empty((rows, num_heads * head_dim), dtype=out_dtype)
    args = capi.GqaPrefillArgs(
        q.data_ptr(), _ptr(k_plane), _ptr(k_scales), _ptr(v_plane), _ptr(v_scales), _ptr(table), out.data_ptr(), None, 0, rows, position,
        window, num_heads, num_kv_heads, head_dim, block_tokens, score_scale, softcap, kv_format, scale_dtype, _DTYPE[q.dtype],
        _DTYPE[out_dtype])
    if gate is not None:
        args.gate, args.gate_cols, args.gate_dtype = gate.data_ptr(), gate.shape[1], _DTYPE[gate.dtype]
    args.visible_ends = _ptr(visible_ends)
    args.visible_starts = _ptr(visible_starts)
    args.table_stride = 0 if table is None else table.numel()
    scratch = None
    if workspace:
        lib = capi.load()
        need = max(lib.zllm_attn_gqa_prefill_preferred_bytes(C.byref(args)), 256)
        scratch = _workspace(need, lib.zllm_attn_gqa_prefill_workspace_bytes, args, q.device)
        args.workspace, args.workspace_bytes = _ptr(scratch), scratch.numel()
    return args, out, scratch


def gqa_prefill_chunk(*a, **kw):
    """One chunk of causal GQA prefill over the paged cache (zllm_attn_gqa_prefill_chunk).  `workspace=False` passes none:
    a chunk that would be cut into KV splits then runs unsplit (geometries that need a workspace fail)."""
    args, out, _scratch = gqa_prefill_chunk_args(*a, **kw)
    capi.check(capi.load().zllm_attn_gqa_prefill_chunk(C.byref(args), _stream()))
    return out


def mla_decode_args(q, kv_b, latent_codes, latent_scales, rope_cache, tables, ctx_lens, heads, q_head_dim,
                    kv_head_dim, latent_dim, rope_dim, block_tokens, max_ctx_len, out_dtype=torch.float32,
                    out_compact=True, out=None, workspace=None, selection=None, selection_counts=None, query_rows=1,
                    total_ctx_tokens=0, wide_tiles=False, kv_b_bits=0, kv_b_scales=None, kv_b_group=0, kv_b_scale_dtype=capi.SCALE_BF16):
    """`q` holds every query row of the call, sequence-major: [batch * query_rows, heads * q_head_dim].
    `kv_b` is bf16 unless kv_b_bits says f32 (32) or packed 8- / 4-bit codes with `kv_b_scales` per `kv_b_group` columns."""
    rows = q.shape[0]
    batch = rows // query_rows
    value_dim = kv_head_dim - (q_head_dim - rope_dim)
    if out is None:
        cols = heads * value_dim if out_compact else heads * q_head_dim
        out = torch.zeros((rows, cols), dtype=out_dtype, device=q.device)
    args = capi.MlaDecodeArgs()
    args.q, args.kv_b, args.latent_codes = _ptr(q), _ptr(kv_b), _ptr(latent_codes)
    args.latent_scales, args.rope_cache = _ptr(latent_scales), _ptr(rope_cache)
    args.tables, args.ctx_lens, args.out = _ptr(tables), _ptr(ctx_lens), _ptr(out)
    args.batch, args.heads, args.q_head_dim, args.kv_head_dim = batch, heads, q_head_dim, kv_head_dim
    args.latent_dim, args.rope_dim = latent_dim, rope_dim
    args.table_stride = 0 if tables is None else tables.shape[1]
    args.max_ctx_len, args.block_tokens = max_ctx_len, block_tokens
    args.q_dtype, args.out_dtype, args.out_compact = _DTYPE[q.dtype], _DTYPE[out_dtype], int(out_compact)
    args.query_rows = query_rows
    args.total_ctx_tokens = total_ctx_tokens
    args.stage_mask = capi.MLA_WIDE_TILES if wide_tiles else 0
    args.kv_b_bits, args.kv_b_scales, args.kv_b_group, args.kv_b_scale_dtype = kv_b_bits, _ptr(kv_b_scales), kv_b_group, kv_b_scale_dtype
    if selection is not None:  # [batch, top_k] token positions (uint32 / int32)
        args.selection, args.top_k = _ptr(selection), selection.shape[1]
        args.selection_counts = _ptr(selection_counts)
    lib = capi.load()
    need = least = lib.zllm_attn_mla_decode_workspace_bytes(C.byref(args))
    if least == 0:
        raise capi.ZllmAttnError(-1, capi.last_error())
    if query_rows > 1 and (workspace is None or workspace.numel() > least):
        need = lib.zllm_attn_mla_decode_preferred_bytes(C.byref(args))
    if workspace is None:
        workspace = _workspace(need, lib.zllm_attn_mla_decode_workspace_bytes, args, q.device)
    args.workspace, args.workspace_bytes = _ptr(workspace), workspace.numel()
    if workspace.numel() >= need > least:  # the number asks for the larger workspace's plan
        args.workspace_bytes = need
    return args, out, workspace


def mla_decode(*a, **kw):
    args, out, workspace = mla_decode_args(*a, **kw)
    capi.check(capi.load().zllm_attn_mla_decode(C.byref(args), _stream()))
    return out


# ---- drafted tokens: a chain or tree of drafts per sequence (node 0 is the token sampled last), verified in a batch --------------

_WORD, _LONG = (torch.int32, torch.uint32), (torch.int64, torch.uint64)


def _words(t, name, count, device, dtypes=_WORD):
    """Address of a contiguous tensor of `count` whole numbers on CUDA device `device` (None: not given)."""
    if t is None:
        return None
    if t.dtype not in dtypes or t.get_device() != device or not t.is_contiguous() or t.numel() != count:
        raise ValueError(f"{name} must be a contiguous tensor of {count} elements of {dtypes[0]} on the call's device (got {tuple(t.shape)} {t.dtype} {t.device})")
    return t.data_ptr()


def _values(t, name, count, device, dtype=None):
    if t is None:
        return None
    if (t.dtype not in _DTYPE if dtype is None else t.dtype != dtype) or t.get_device() != device or not t.is_contiguous() or t.numel() != count:
        raise ValueError(f"{name} must be a contiguous tensor of {count} elements of {dtype or 'f32, bf16 or f16'} on the call's device "
                         f"(got {tuple(t.shape)} {t.dtype} {t.device})")
    return t.data_ptr()


def _plane(t, name, device):
    if t is None:
        return None
    if t.get_device() != device or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous tensor on the call's device")
    return t.data_ptr()


_CODES, _HALVES = (torch.int8, torch.uint8), (torch.float16,)
_SCALES = {capi.SCALE_BF16: torch.bfloat16, capi.SCALE_F16: torch.float16, capi.SCALE_F32: torch.float32}
_RULE_SCALES = {capi.QUANT_ROCM_MLA: torch.bfloat16, capi.QUANT_METAL_GQA: torch.float16, capi.QUANT_CUDA_GQA: torch.float32, capi.QUANT_RECIPROCAL_GQA: torch.float16}


def _rows_of(plane, name, cols, dtypes, device):
    """Address and size of a plane of rows of `cols` elements (None: not given, which the C call says)."""
    if plane is None:
        return None, 0
    count = plane.numel()
    if plane.dtype not in dtypes or count == 0 or count % cols != 0 or plane.get_device() != device or not plane.is_contiguous():
        raise ValueError(f"{name} must be a contiguous tensor of rows of {cols} {dtypes[0]} on the call's device (got {tuple(plane.shape)} {plane.dtype} {plane.device})")
    return plane.data_ptr(), count


def _scales_of(scales, name, codes, dtype, device):
    if scales is None:
        return None
    if (scales.dtype != dtype and dtype is not None) or (codes != 0 and scales.numel() * 64 != codes) or scales.get_device() != device or not scales.is_contiguous():
        raise ValueError(f"{name} must be a contiguous tensor of {dtype}, one for every 64 codes of its plane, on the call's device (got {tuple(scales.shape)} {scales.dtype} {scales.device})")
    return scales.data_ptr()


def _cache_planes(k_plane, k_scales, v_plane, v_scales, num_kv_heads, head_dim, kv_format, scales, device):
    """Addresses of a cache's planes: rows of num_kv_heads * head_dim int8 codes with a scale of type `scales` (None: any) per 64, or of f16 values."""
    cols = max(num_kv_heads * head_dim, 1)
    if kv_format == capi.KV_F16:
        return _rows_of(k_plane, "k_plane", cols, _HALVES, device)[0], None, _rows_of(v_plane, "v_plane", cols, _HALVES, device)[0], None
    k, k_codes = _rows_of(k_plane, "k_plane", cols, _CODES, device)
    v, v_codes = _rows_of(v_plane, "v_plane", cols, _CODES, device)
    return k, _scales_of(k_scales, "k_scales", k_codes, scales, device), v, _scales_of(v_scales, "v_scales", v_codes, scales, device)


def _current(t, name):
    """The current device, which is where the call's tensors have to be."""
    device = torch.cuda.current_device() if t.is_cuda else -1
    if t.get_device() != device or device < 0:
        raise ValueError(f"{name} on {t.device}: the call's tensors must be on the current CUDA device")
    return device


def _sequences(q, tables):
    """The device, q's rows, the sequences, rows a sequence and pages a table of a call on q [batch * rows, ...] and tables [batch, pages]."""
    nodes, shape = q.shape[0], tables.shape
    batch = shape[0]
    rows = nodes // max(batch, 1)
    if rows * batch != nodes or len(shape) != 2:
        raise ValueError(f"q has {nodes} rows and tables {tuple(shape)}: not the same number of rows a sequence")
    return _current(q, "q"), nodes, batch, rows, shape[1]


def _stream_of(device):
    return torch.cuda.current_stream().cuda_stream if _raw_stream is None else _raw_stream(device)


def draft_layout(parents, kv_lens, row_counts=None):
    """Ancestor masks int64 [batch, rows, ceil(rows / 64)] and token positions int32 [batch, rows] of the trees that `parents`
    int32 [batch, rows] describes (-1: none) (zllm_attn_draft_layout)."""
    device = _current(parents, "parents")
    batch, rows = parents.shape
    masks = parents.new_empty((batch, rows, (rows + 63) // 64), dtype=torch.int64)
    positions = torch.empty_like(parents, dtype=torch.int32)
    args = capi.DraftLayoutArgs(_words(parents, "parents", batch * rows, device), _words(kv_lens, "kv_lens", batch, device),
                                _words(row_counts, "row_counts", batch, device), masks.data_ptr(), positions.data_ptr(), batch, rows)
    capi.check(capi.load().zllm_attn_draft_layout(C.byref(args), _stream_of(device)))
    return masks, positions


def gqa_draft_prologue(q, k, v, q_norm, k_norm, cos, sin, k_plane, k_scales, v_plane, v_scales, tables, kv_lens, num_heads, num_kv_heads, head_dim,
                       rotary_dim, block_tokens, positions=None, row_counts=None, eps=1e-6, weight_offset=1.0, rule=capi.QUANT_RECIPROCAL_GQA, split_half=True,
                       q_out_dtype=torch.float32, kv_format=capi.KV_Q8G64, ring_capacity=0):
    """gqa_prologue for the drafted nodes of a batch: q [batch * rows, heads * dim]; node i of sequence b rotates at positions[b, i] and its K
    and V go to cache token kv_lens[b] + i (zllm_attn_gqa_draft_prologue).  By default the Q8g64 rows are those that the formula gives as a torch program on
    the device, bit for bit; `rule` names that of the cache's other rows where a node must have the bits gqa_prologue (METAL_GQA by default) would write."""
    device, nodes, batch, rows, stride = _sequences(q, tables)
    q_out = q.new_empty((nodes, num_heads * head_dim), dtype=q_out_dtype)
    angles = 0 if cos is None else cos.shape[0]
    args = capi.GqaDraftPrologueArgs(
        _values(q, "q", nodes * num_heads * head_dim, device), _values(k, "k", nodes * num_kv_heads * head_dim, device, q.dtype),
        _values(v, "v", nodes * num_kv_heads * head_dim, device, q.dtype), _values(q_norm, "q_norm", head_dim, device, torch.float32),
        _values(k_norm, "k_norm", head_dim, device, torch.float32), _values(cos, "cos", angles * (rotary_dim // 2), device, torch.float32),
        _values(sin, "sin", angles * (rotary_dim // 2), device, torch.float32), q_out.data_ptr(),
        *_cache_planes(k_plane, k_scales, v_plane, v_scales, num_kv_heads, head_dim, kv_format, _RULE_SCALES.get(rule), device), _words(tables, "tables", batch * stride, device),
        _words(kv_lens, "kv_lens", batch, device), _words(positions, "positions", nodes, device), _words(row_counts, "row_counts", batch, device), batch, rows, num_heads,
        num_kv_heads, head_dim, rotary_dim, angles, stride, block_tokens, ring_capacity, eps, weight_offset, _DTYPE[q.dtype], _DTYPE[q_out_dtype],
        kv_format, rule, int(split_half))
    capi.check(capi.load().zllm_attn_gqa_draft_prologue(C.byref(args), _stream_of(device)))
    return q_out


def gqa_draft_attention_args(q, k_plane, k_scales, v_plane, v_scales, tables, kv_lens, masks, num_heads, num_kv_heads, head_dim, block_tokens, score_scale,
                             max_kv_len, positions=None, row_counts=None, window=0, softcap=0.0, ring_capacity=0, kv_format=capi.KV_Q8G64,
                             scale_dtype=capi.SCALE_F16, out_dtype=torch.float32, out=None, workspace=None, total_kv_tokens=0, gate=None):
    """The argument block of zllm_attn_gqa_draft_attention, the output tensor and the workspace tensor: for callers that launch the same call many
    times."""
    device, nodes, batch, rows, stride = _sequences(q, tables)
    if out is None:
        out = q.new_empty((nodes, num_heads * head_dim), dtype=out_dtype)
    args = capi.GqaDraftAttentionArgs(
        _values(q, "q", nodes * num_heads * head_dim, device),
        *_cache_planes(k_plane, k_scales, v_plane, v_scales, num_kv_heads, head_dim, kv_format, _SCALES.get(scale_dtype), device), _words(tables, "tables", batch * stride, device), _words(kv_lens, "kv_lens", batch, device),
        _words(masks, "masks", nodes * ((rows + 63) // 64), device, _LONG), _words(positions, "positions", nodes, device), _words(row_counts, "row_counts", batch, device),
        _values(out, "out", nodes * num_heads * head_dim, device), None, 0, batch, rows, num_heads, num_kv_heads, head_dim, stride, max_kv_len, total_kv_tokens,
        block_tokens, ring_capacity, window, score_scale, softcap, kv_format, scale_dtype, _DTYPE[q.dtype], _DTYPE[out.dtype])
    if gate is not None:
        if gate.dim() != 2:
            raise ValueError(f"gate must be [{nodes}, 1 or {num_heads * head_dim}] (got {tuple(gate.shape)})")
        args.gate, args.gate_cols, args.gate_dtype = _values(gate, "gate", nodes * gate.shape[1], device), gate.shape[1], _DTYPE[gate.dtype]
    if workspace is None:
        need = capi.load().zllm_attn_gqa_draft_attention_workspace_bytes(C.byref(args))
        if need == 0:
            raise capi.ZllmAttnError(-1, capi.last_error())
        workspace = q.new_empty(need, dtype=torch.uint8)
        args.workspace, args.workspace_bytes = workspace.data_ptr(), need
    else:
        args.workspace, args.workspace_bytes = _plane(workspace, "workspace", device), workspace.numel() * workspace.element_size()
    return args, out, workspace


def gqa_draft_attention(q, *a, **kw):
    """Attention of the drafted nodes of a batch, q [batch * rows, heads * dim]: node i of sequence b attends the sequence's kv_lens[b] cached tokens
    and the nodes that masks[b, i] names (None: a chain) (zllm_attn_gqa_draft_attention)."""
    args, out, _workspace_tensor = gqa_draft_attention_args(q, *a, **kw)
    capi.check(capi.load().zllm_attn_gqa_draft_attention(C.byref(args), _stream_of(q.get_device())))
    return out


def _prob_rows(t, name, rows, vocab, device):
    """A tensor of `rows` distributions, [..., vocab] with evenly spaced rows that do not overlap: its elements from row to row."""
    if t.dtype not in _DTYPE or t.get_device() != device or t.shape[-1] != vocab or t.numel() != rows * vocab or (vocab > 1 and t.stride(-1) != 1):
        raise ValueError(f"{name} must be {rows} rows of {vocab} f32, bf16 or f16 values on the call's device (got {tuple(t.shape)} {t.dtype} {t.device})")
    if t.is_contiguous():
        return vocab
    spaced = [(t.shape[i], t.stride(i)) for i in range(t.dim() - 1) if t.shape[i] > 1]
    for (_, outer), (count, inner) in zip(spaced, spaced[1:]):
        if outer != inner * count:
            raise ValueError(f"{name}: rows must be evenly spaced")
    stride = spaced[-1][1] if spaced else vocab
    if stride < vocab:
        raise ValueError(f"{name}: rows must not overlap (expanded tensors: call contiguous() first)")
    return stride


def draft_verify(tokens, target_probs, uniforms, parents=None, draft_probs=None, row_counts=None, workspace=None):
    """Accepts drafts (tokens int32 [batch, rows]) against target_probs [batch, rows, vocab] from given uniforms f32 [batch, rows]; draft_probs
    [batch, rows - 1, vocab] where a chain's drafts were drawn from distributions.  Returns path, accepted and out_tokens
    (zllm_attn_draft_verify)."""
    device = _current(target_probs, "target_probs")
    batch, rows = tokens.shape
    vocab = target_probs.shape[-1]
    target_stride = _prob_rows(target_probs, "target_probs", batch * rows, vocab, device)
    draft_stride = 0
    if draft_probs is not None and rows == 1:
        draft_probs = None  # no drafts
    if draft_probs is not None:
        draft_stride = _prob_rows(draft_probs, "draft_probs", batch * (rows - 1), vocab, device)
    path, out_tokens = torch.empty_like(tokens, dtype=torch.int32), torch.empty_like(tokens, dtype=torch.int32)
    accepted = tokens.new_empty(batch, dtype=torch.int32)
    args = capi.DraftVerifyArgs(
        _words(tokens, "tokens", batch * rows, device), _words(parents, "parents", batch * rows, device), _words(row_counts, "row_counts", batch, device), target_probs.data_ptr(),
        _ptr(draft_probs), _values(uniforms, "uniforms", batch * rows, device, torch.float32), path.data_ptr(), accepted.data_ptr(), out_tokens.data_ptr(), None, 0,
        target_stride, draft_stride, batch, rows, vocab, _DTYPE[target_probs.dtype], 0 if draft_probs is None else _DTYPE[draft_probs.dtype])
    lib = capi.load()
    if workspace is None:
        need = lib.zllm_attn_draft_verify_workspace_bytes(C.byref(args))
        if need == 0:
            raise capi.ZllmAttnError(-1, capi.last_error())
        workspace = torch.empty(need, dtype=torch.uint8, device=tokens.device)
    args.workspace, args.workspace_bytes = _plane(workspace, "workspace", device), workspace.numel() * workspace.element_size()
    capi.check(lib.zllm_attn_draft_verify(C.byref(args), _stream_of(device)))
    return path, accepted, out_tokens


def _commit_plane(t, device):
    """Bytes of a row of a plane [rows, columns]."""
    _plane(t, "a plane", device)
    if t.dim() != 2:
        raise ValueError(f"a plane must be [rows, columns], a row a token (got {tuple(t.shape)})")
    return t.shape[1] * t.element_size()


class CommitPlanes:
    """The planes of a cache (tensors of one row a token) as zllm_attn_commit_rows reads them: made once, used every step."""

    def __init__(self, planes):
        planes = list(planes)
        if not planes:
            raise ValueError("no planes")
        self.device = _current(planes[0], "a plane")
        row_bytes = [_commit_plane(plane, self.device) for plane in planes]
        if len({t.data_ptr() for t in planes}) != len(planes):
            raise ValueError("a plane is given twice: its rows would move twice")
        self.tensors = planes
        self.array = (capi.KvPlane * len(planes))(*[capi.KvPlane(t.data_ptr(), size) for t, size in zip(planes, row_bytes)])


def commit_planes(planes):
    return CommitPlanes(planes)


def commit_rows(planes, tables, kv_lens, path, accepted, block_tokens, ring_capacity=0):
    """Moves the accepted nodes' rows behind the sequences' tokens in every plane of `planes` (commit_planes(...), or a list of planes); returns the
    new lengths int32 [batch] (zllm_attn_commit_rows)."""
    if not isinstance(planes, CommitPlanes):
        planes = CommitPlanes(planes)
    device = planes.device
    batch, rows = path.shape
    new_lens = kv_lens.new_empty(batch, dtype=torch.int32)
    args = capi.CommitRowsArgs(planes.array, _words(tables, "tables", batch * tables.shape[1], device), _words(kv_lens, "kv_lens", batch, device),
                               _words(path, "path", batch * rows, device), _words(accepted, "accepted", batch, device), new_lens.data_ptr(), len(planes.tensors), batch, rows,
                               tables.shape[1], block_tokens, ring_capacity)
    capi.check(capi.load().zllm_attn_commit_rows(C.byref(args), _stream_of(_current(path, "path"))))
    return new_lens
