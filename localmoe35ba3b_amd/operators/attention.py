"""Attention between the MoE blocks: norms of queries and keys with the position
rotation, a paged cache of keys and values, and attention over it.

qk_norm_rope      per-head RMSNorm (scale 1 + w) and rotation of queries and keys
append            keys (normed and rotated on the way) and values into the cache,
                  with the queries of the same tokens in the same pass
paged_attention   each sequence's new tokens over its cache, causal at its end

A cache is two tensors [pages, kv_heads, page_size, head_dim], keys and values.  A
batch is three int32 tensors on the GPU, which a program keeps for all layers of a
step and may rewrite between replays of a captured step:
  starts  [sequences + 1]  the rows of sequence s are starts[s] .. starts[s + 1] - 1
  lengths [sequences]      its positions, the new ones (its last) among them
  table   [sequences, n]   the page of its positions i * page_size ..
Rows of no sequence (padding behind the last) are left as they were.

The reference has no operators of this kind (its layers run the Transformers
modules, HF:627-735).
"""
import torch

from .. import _lib

_TYPES = (torch.bfloat16, torch.float16)


def _rows(x, what):
    """x [tokens, heads, head_dim] with contiguous, 16-byte aligned heads; a copy of others."""
    if not x.is_cuda or x.ndim != 3 or x.dtype not in _TYPES:
        raise ValueError(f'{what}: expected CUDA FP16/BF16 rows [tokens, heads, head_dim]')
    token, head, channel = x.stride()
    if channel != 1 or token % 8 or head % 8 or x.data_ptr() % 16:
        x = x.contiguous()
        if x.data_ptr() % 16:
            x = x.clone()
    return x


def _weight(w, x):
    """fp32 norm weights on the device of x, or None."""
    if w is None:
        return None
    if w.numel() != x.shape[-1]:
        raise ValueError('norm weight does not match the head size')
    if w.dtype is not torch.float32 or w.device != x.device or not w.is_contiguous():
        w = w.to(device=x.device, dtype=torch.float32).contiguous()
    return w if w.data_ptr() % 16 == 0 else w.clone()


def _frequencies(inv_freq, x):
    """fp32 frequencies on the device of x, or None, and how many."""
    if inv_freq is None:
        return None, 0
    pairs = inv_freq.numel()
    if pairs < 8 or pairs % 8 or 2 * pairs > x.shape[-1]:
        raise ValueError('rotated channels must be a multiple of 16 and fit the head')
    if (inv_freq.dtype is not torch.float32 or inv_freq.device != x.device
            or not inv_freq.is_contiguous()):
        inv_freq = inv_freq.to(device=x.device, dtype=torch.float32).contiguous()
    return inv_freq, pairs


def _same(x, *others):
    for o in others:
        if o.dtype is not x.dtype or o.device != x.device:
            raise ValueError('attention tensors must share their type and device')


def qk_norm_rope(q, k, q_weight, k_weight, positions, inv_freq, eps=1e-6):
    """Normed and rotated (q, k), contiguous [tokens, heads, head_dim] each.

    q [T, q_heads, D], k [T, k_heads, D] (bf16 or fp16, D = 64, 128 or 256, any token
    and head strides); weights [D] (scale 1 + w) or None for no norm; positions int64
    [T]; inv_freq [R / 2] rotates channels i and i + R / 2 by positions * inv_freq[i]
    (None: no rotation)."""
    q, k = _rows(q, 'queries'), _rows(k, 'keys')
    _same(q, k)
    tokens, q_heads, dim = q.shape
    k_heads = k.shape[1]
    if k.shape[0] != tokens or k.shape[2] != dim:
        raise ValueError('queries and keys do not match')
    if positions.device != q.device or positions.numel() != tokens:
        raise ValueError('Expected a CUDA position of every token')
    positions = positions.to(torch.int64).contiguous()
    q_weight, k_weight = _weight(q_weight, q), _weight(k_weight, k)
    inv_freq, pairs = _frequencies(inv_freq, q)
    q_out, k_out = q.new_empty((tokens, q_heads, dim)), k.new_empty((tokens, k_heads, dim))
    _lib.call_on(q.device, 'lm_qk_norm_rope', q.data_ptr(), q.stride(0), q.stride(1), q_heads,
              _lib.ptr(q_weight), q_out.data_ptr(), k.data_ptr(), k.stride(0), k.stride(1),
              k_heads, _lib.ptr(k_weight), k_out.data_ptr(), positions.data_ptr(),
              _lib.ptr(inv_freq), pairs, tokens, dim, eps, _lib.dtype_code(q.dtype),
              _lib.stream(q.device))
    return q_out, k_out


def _cache(k_pages, v_pages):
    """(pages, page stride, kv_heads, page_size, head_dim) of a cache."""
    if (k_pages.ndim != 4 or k_pages.shape != v_pages.shape or not k_pages.is_cuda
            or k_pages.dtype not in _TYPES or k_pages.stride() != v_pages.stride()):
        raise ValueError('Expected CUDA key and value pages [pages, kv_heads, page_size, head_dim]')
    _same(k_pages, v_pages)
    pages, heads, size, dim = k_pages.shape
    stride, *inner = k_pages.stride()
    if tuple(inner) != (size * dim, dim, 1):
        raise ValueError('the values of a page must be contiguous')
    return pages, stride if pages > 1 else heads * size * dim, heads, size, dim


def _batch(device, starts, lengths, table):
    """The C arguments of a batch: pointers, table stride, table pages, sequences."""
    for t in (starts, lengths, table):
        if t.dtype is not torch.int32 or t.device != device:
            raise ValueError('Expected CUDA int32 starts, lengths and page table')
    sequences = lengths.numel()
    if starts.numel() != sequences + 1 or table.ndim != 2 or table.shape[0] != sequences:
        raise ValueError('starts, lengths and page table do not match')
    if not (starts.is_contiguous() and lengths.is_contiguous()) or (
            table.shape[1] > 1 and table.stride(1) != 1):
        raise ValueError('starts, lengths and the rows of the page table must be contiguous')
    return (starts.data_ptr(), lengths.data_ptr(), table.data_ptr(),
            table.stride(0) if sequences > 1 else table.shape[1], table.shape[1], sequences)


def append(k_pages, v_pages, k, v, starts, lengths, table, inv_freq=None, k_weight=None, q=None,
           q_weight=None, eps=1e-6):
    """Appends k and v [T, kv_heads, D] to the cache, k normed and rotated on the way
    (k_weight and inv_freq as in qk_norm_rope, by its position in its sequence).
    With q [T, q_heads, D], returns the queries normed and rotated for
    paged_attention; rows of no sequence are not written there."""
    pages, stride, heads, size, dim = _cache(k_pages, v_pages)
    k, v = _rows(k, 'keys'), _rows(v, 'values')
    _same(k_pages, k, v)
    tokens = k.shape[0]
    if k.shape != v.shape or k.shape[1] != heads or k.shape[2] != dim:
        raise ValueError('keys and values do not match the cache')
    q_args = (None, 0, 0, 0, None, None)
    q_out = None
    if q is not None:
        q = _rows(q, 'queries')
        _same(k, q)
        if q.shape[0] != tokens or q.shape[2] != dim:
            raise ValueError('queries and keys do not match')
        q_weight = _weight(q_weight, q)
        q_out = q.new_empty(q.shape)
        q_args = (q.data_ptr(), q.stride(0), q.stride(1), q.shape[1], _lib.ptr(q_weight),
                  q_out.data_ptr())
    k_weight = _weight(k_weight, k)
    inv_freq, pairs = _frequencies(inv_freq, k)
    batch = _batch(k.device, starts, lengths, table)
    _lib.call_on(k.device, 'lm_paged_append', k.data_ptr(), k.stride(0), k.stride(1), _lib.ptr(k_weight),
              v.data_ptr(), v.stride(0), v.stride(1), *q_args, k_pages.data_ptr(),
              v_pages.data_ptr(), pages, stride, heads, size, dim, *batch, _lib.ptr(inv_freq),
              pairs, tokens, eps, _lib.dtype_code(k.dtype), _lib.stream(k.device))
    return q_out


def paged_attention(q, k_pages, v_pages, starts, lengths, table, scale=None, gate=None,
                    max_new=None, out=None):
    """Attention of the new tokens q [T, q_heads, D] over the cache -> [T, q_heads, D].

    The token at position p of its sequence sees the positions up to p.  scale
    defaults to D ** -0.5; gate [T, q_heads, D] multiplies the result by sigmoid(gate).
    max_new bounds the new tokens of one sequence (default: T); a close bound saves
    time.  out [T, q_heads, D], contiguous, receives the result; rows of no sequence
    keep what they hold there."""
    pages, stride, heads, size, dim = _cache(k_pages, v_pages)
    q = _rows(q, 'queries')
    _same(k_pages, q)
    tokens, q_heads = q.shape[:2]
    if q.shape[2] != dim or q_heads % heads:
        raise ValueError('queries do not match the cache')
    gate_args = (None, 0, 0)
    if gate is not None:
        gate = _rows(gate, 'gate')
        _same(q, gate)
        if gate.shape != q.shape:
            raise ValueError('gate does not match the queries')
        gate_args = (gate.data_ptr(), gate.stride(0), gate.stride(1))
    if out is None:
        out = q.new_empty(q.shape)
    else:
        _same(q, out)
        if out.shape != q.shape or not out.is_contiguous() or out.data_ptr() % 16:
            raise ValueError('Expected a contiguous output of the shape of the queries')
    batch = _batch(q.device, starts, lengths, table)
    max_new = tokens if max_new is None else max_new
    need = _lib.lib().lm_paged_attention_workspace_bytes(tokens, batch[5], q_heads, heads, dim,
                                                         max_new, batch[4] * size)
    workspace = q.new_empty(need, dtype=torch.uint8) if need > 0 else None
    _lib.call_on(q.device, 'lm_paged_attention', q.data_ptr(), q.stride(0), q.stride(1), q_heads,
              k_pages.data_ptr(), v_pages.data_ptr(), pages, stride, heads, size, dim, *batch,
              tokens, max_new, dim ** -0.5 if scale is None else scale, *gate_args,
              out.data_ptr(), _lib.ptr(workspace), need, _lib.dtype_code(q.dtype),
              _lib.stream(q.device))
    return out
