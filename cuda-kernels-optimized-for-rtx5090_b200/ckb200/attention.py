"""Paged attention on B200: run({"q", "key_cache", "value_cache", "block_tables", "seq_lens"[, "scale", "shared_prefix"]})
-> {"out"}.

The attention of a decoding step over the cache that rope.rope_kv_cache and rope.qk_norm_rope_kv_cache write: one new token
of each sequence, or several drafted ones, grouped query heads, and a prefix (a system prompt, a document) that all
sequences of the batch share and that is then read once for the whole batch. No counterpart in the reference; the
library's C entry is ckb_attention_paged_launch.
"""

import struct

import torch

from . import _native

_DTYPES = {torch.bfloat16: 1, torch.float16: 2}
_STRIDES = struct.Struct("3q")
_needs = {}  # (device, sizes) -> bytes of workspace


def _problem(q, key_cache, value_cache, tables, lens, prefix):
    """Why these inputs are not an attention these kernels serve, or None."""
    q_shape, shape, dtype = q.shape, key_cache.shape, q.dtype
    if dtype not in _DTYPES or len(q_shape) != 4 or q_shape[1] < 1 or q_shape[2] < 1 or q_shape[3] < 1:
        return f"q {dtype} {tuple(q_shape)}, bf16 or fp16 [B, T, Hq, D] is served"
    batch, _, q_heads, head_dim = q_shape
    if head_dim % 8 or head_dim > 256:
        return f"head_dim {head_dim}, a multiple of 8 up to 256 is served"
    if shape != value_cache.shape:
        return f"key_cache {tuple(shape)} and value_cache {tuple(value_cache.shape)} differ"
    for name, c in (("key_cache", key_cache), ("value_cache", value_cache)):
        if c.dtype != dtype or len(shape) != 4 or shape[3] != head_dim or shape[1] < 1 or shape[2] < 1 or \
                not c.is_contiguous():
            return (f"{name} must be a contiguous [blocks, block_size, Hkv, {head_dim}] tensor of {dtype}, got {c.dtype} "
                    f"{tuple(shape)}")
    if q_heads % shape[2]:
        return f"{q_heads} query heads for {shape[2]} key heads"
    if tables.dtype != torch.int64 or tables.dim() != 2 or tables.shape[0] != batch or tables.shape[1] < 1:
        return f"block_tables {tables.dtype} {tuple(tables.shape)}, int64 [{batch}, blocks] is needed"
    if lens.dtype != torch.int64 or lens.shape != (batch,):
        return f"seq_lens {lens.dtype} {tuple(lens.shape)}, int64 [{batch}] is needed"
    block_size = shape[1]
    if not isinstance(prefix, int) or prefix < 0 or prefix % block_size or prefix > tables.shape[1] * block_size:
        return (f"shared_prefix {prefix!r} must be a number of tokens, a multiple of the block size {block_size}, within the "
                f"{tables.shape[1]} blocks of a sequence")
    return None


def paged_attention(q, key_cache, value_cache, block_tables, seq_lens, scale=None, shared_prefix=0, out=None):
    """softmax(scale * q k^T) v over each sequence's cached tokens: [B, T, Hq, D] in q's dtype.

    q [B, T, Hq, D] (bf16 or fp16, any strides with a contiguous last dim, so a view of a fused projection) holds the T
    newest tokens of each sequence, whose keys and values are in the cache already; key_cache / value_cache [num_blocks,
    block_size, Hkv, D] in the same dtype; block_tables [B, M] int64, the blocks of each sequence in order; seq_lens [B]
    int64, the tokens of each sequence with the T new ones. Token t sees the positions below seq_lens - T + t + 1; with
    none (a padded row of the batch: length 0) its output is zeros. scale defaults to D ** -0.5. shared_prefix: the number
    of tokens (a multiple of block_size) with which the sequences begin in the SAME blocks; they are read once, through the
    block_tables row of the first sequence all of whose T tokens see them all. Sequences that end before that (padded rows
    among them) are read through their own rows, so a row's entries behind its length are never looked at. A block id
    outside the cache reads as zeros. Scores, softmax statistics and sums are fp32."""
    problem = _problem(q, key_cache, value_cache, block_tables, seq_lens, shared_prefix)
    if problem:
        raise ValueError(f"attention: {problem}")
    batch, tokens, q_heads, head_dim = q.shape
    scale = head_dim ** -0.5 if scale is None else float(scale)
    if not 0.0 < scale < 1e30:
        raise ValueError(f"attention: scale must be a positive finite number, got {scale}")
    _native.require_cuda("attention", q, key_cache, value_cache, block_tables, seq_lens)
    if key_cache.data_ptr() % 16 or value_cache.data_ptr() % 16:
        raise ValueError("attention: the caches must start on 16-byte boundaries")
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    elif out.shape != q.shape or out.dtype != q.dtype or not out.is_contiguous() or out.device != q.device or \
            out.data_ptr() % 16:
        raise ValueError("attention: out must be a contiguous, 16-byte aligned tensor of q's shape, dtype and device")
    if batch == 0:
        return out
    st_b, st_t, st_h, st_d = q.stride()
    st_b, st_t, st_h = 0 if batch == 1 else st_b, 0 if tokens == 1 else st_t, 0 if q_heads == 1 else st_h
    if st_d != 1 or st_b % 8 or st_t % 8 or st_h % 8 or q.data_ptr() % 16:
        q = q.clone(memory_format=torch.contiguous_format)
        st_b, st_t, st_h, _ = q.stride()
    tables, lens = block_tables.contiguous(), seq_lens.contiguous()
    num_blocks, block_size, kv_heads, _ = key_cache.shape
    width = tables.shape[1]
    lib = _native.load("attention")
    sizes = (batch, tokens, q_heads, kv_heads, head_dim, block_size, width, shared_prefix)
    key = (q.get_device(), sizes)
    need = _needs.get(key)
    if need is None:
        need = _native.on_device(lib.ckb_attention_workspace, q, *sizes)
        if need < 0:
            raise ValueError(f"attention: sizes beyond what is served: q {tuple(q.shape)}, caches {tuple(key_cache.shape)}, "
                             f"block_tables {tuple(tables.shape)}")
        if len(_needs) > 256:
            _needs.clear()
        _needs[key] = need
    work = q.new_empty((need,), dtype=torch.uint8)
    _native.call(lib.ckb_attention_paged_launch, q, q.data_ptr(), key_cache.data_ptr(), value_cache.data_ptr(),
                 tables.data_ptr(), lens.data_ptr(), out.data_ptr(), work.data_ptr(), need, _STRIDES.pack(st_b, st_t, st_h),
                 batch, tokens, q_heads, kv_heads, head_dim, num_blocks, block_size, width, shared_prefix, scale,
                 _DTYPES[q.dtype])
    return out


def check(device=None):
    """Synchronises the device (by default the current one) and raises RuntimeError when a wait of these kernels on a copy or a
    product has run out there since the last check: every wait ends after 2 s at most, and outputs of the calls since then
    may be void."""
    lib = _native.load("attention")
    if device is None:
        status = lib.ckb_attention_status(1)
    else:
        with torch.cuda.device(device):
            status = lib.ckb_attention_status(1)
    if status < 0:
        raise RuntimeError(f"attention: status read failed: CUDA error {-status}")
    if status:
        raise RuntimeError("attention: a wait inside a kernel ran out (2 s); the outputs since the last check may be void")


def run(inputs):
    return {"out": paged_attention(inputs["q"], inputs["key_cache"], inputs["value_cache"], inputs["block_tables"],
                                   inputs["seq_lens"], inputs.get("scale"), inputs.get("shared_prefix", 0))}
