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
Rows of no sequence (padding behind the last) touch neither the cache nor an output
that the caller gave.

The reference has no operators of this kind (its layers run the Transformers
modules, HF:627-735).
"""
import functools

import torch

from .. import _lib

_TYPES = (torch.bfloat16, torch.float16)


def _rows(x, what):
    """x [tokens, heads, head_dim] with contiguous, 16-byte aligned heads (a copy of others),
    and its strides."""
    if not x.is_cuda or x.ndim != 3 or x.dtype not in _TYPES:
        raise ValueError(f'{what}: expected CUDA FP16/BF16 rows [tokens, heads, head_dim]')
    token, head, channel = x.stride()
    if channel != 1 or token % 8 or head % 8 or x.data_ptr() % 16:
        x = x.contiguous()
        if x.data_ptr() % 16:
            x = x.clone()
        # not x.stride(): torch calls one token or one head contiguous whatever its stride is
        _, heads, dim = x.shape
        token, head = heads * dim, dim
    return x, token, head


def _same(x, dtype, device):
    if x.dtype is not dtype or x.get_device() != device:
        raise ValueError('attention tensors must share their type and device')


def _weight(w, dim, device):
    """fp32 norm weights [dim] on the device, 16-byte aligned, and their address (0: no norm)."""
    if w is None:
        return None, 0
    if w.numel() != dim:
        raise ValueError('norm weight does not match the head size')
    if w.dtype is not torch.float32 or w.get_device() != device or not w.is_contiguous():
        w = w.to(device=device, dtype=torch.float32).contiguous()
    at = w.data_ptr()
    if at % 16:
        w = w.clone()
        at = w.data_ptr()
    return w, at


def check_frequencies(inv_freq, dim):
    """The rotated pairs of heads of `dim`, 0 without a rotation; raises where the operators do."""
    if inv_freq is None:
        return 0
    pairs = inv_freq.numel()
    if pairs < 8 or pairs % 8 or 2 * pairs > dim:
        raise ValueError('rotated channels must be a multiple of 16 and fit the head')
    return pairs


def _frequencies(inv_freq, dim, device):
    """fp32 frequencies on the device, their address (0: no rotation), and how many."""
    pairs = check_frequencies(inv_freq, dim)
    if not pairs:
        return None, 0, 0
    if (inv_freq.dtype is not torch.float32 or inv_freq.get_device() != device
            or not inv_freq.is_contiguous()):
        inv_freq = inv_freq.to(device=device, dtype=torch.float32).contiguous()
    return inv_freq, inv_freq.data_ptr(), pairs


def qk_norm_rope(q, k, q_weight, k_weight, positions, inv_freq, eps=1e-6):
    """Normed and rotated (q, k), contiguous [tokens, heads, head_dim] each.

    q [T, q_heads, D], k [T, k_heads, D] (bf16 or fp16, D = 64, 128 or 256, any token
    and head strides); weights [D] (scale 1 + w) or None for no norm; positions int64
    [T]; inv_freq [R / 2] rotates channels i and i + R / 2 by positions * inv_freq[i]
    (None: no rotation)."""
    q, q_token, q_head = _rows(q, 'queries')
    k, k_token, k_head = _rows(k, 'keys')
    dtype, device = q.dtype, q.get_device()
    _same(k, dtype, device)
    tokens, q_heads, dim = q.shape
    k_tokens, k_heads, k_dim = k.shape
    if k_tokens != tokens or k_dim != dim:
        raise ValueError('queries and keys do not match')
    if positions.get_device() != device or positions.numel() != tokens:
        raise ValueError('Expected a CUDA position of every token')
    if positions.dtype is not torch.int64 or not positions.is_contiguous():
        positions = positions.to(torch.int64).contiguous()
    q_weight, q_w = _weight(q_weight, dim, device)
    k_weight, k_w = _weight(k_weight, dim, device)
    inv_freq, freq, pairs = _frequencies(inv_freq, dim, device)
    q_out, k_out = q.new_empty((tokens, q_heads, dim)), k.new_empty((tokens, k_heads, dim))
    _lib.launch(device, 'lm_qk_norm_rope', q.data_ptr(), q_token, q_head, q_heads, q_w,
                q_out.data_ptr(), k.data_ptr(), k_token, k_head, k_heads, k_w, k_out.data_ptr(),
                positions.data_ptr(), freq, pairs, tokens, dim, eps, _lib.dtype_code(dtype))
    return q_out, k_out


def _cache(k_pages, v_pages, dtype, device):
    """(pages, page stride, kv_heads, page_size, head_dim) of a cache."""
    shape, strides = k_pages.shape, k_pages.stride()
    if len(shape) != 4 or v_pages.shape != shape:
        raise ValueError('Expected key and value pages [pages, kv_heads, page_size, head_dim]')
    _same(k_pages, dtype, device)
    _same(v_pages, dtype, device)
    pages, heads, size, dim = shape
    if heads < 1:
        raise ValueError('Expected pages with key-value heads')
    if strides[1:] != (size * dim, dim, 1) or v_pages.stride() != strides:
        # the stride of a dimension of size 1 is of no consequence
        strides, other = _page_strides(k_pages), _page_strides(v_pages)
        if strides != other:
            raise ValueError('key and value pages must lie alike')
        if strides[1:] != (size * dim, dim, 1):
            raise ValueError('the values of a page must be contiguous')
    return pages, strides[0] if pages > 1 else heads * size * dim, heads, size, dim


def _page_strides(x):
    """Strides, of dimensions of size 1 those of contiguous pages."""
    _, heads, size, dim = x.shape
    plain = heads * size * dim, size * dim, dim, 1
    return tuple(p if n == 1 else s for n, s, p in zip(x.shape, x.stride(), plain))


def _batch(device, starts, lengths, table):
    """The C arguments of a batch: pointers, table stride, table pages, sequences."""
    i32 = torch.int32
    if (starts.dtype is not i32 or lengths.dtype is not i32 or table.dtype is not i32
            or starts.get_device() != device or lengths.get_device() != device
            or table.get_device() != device):
        raise ValueError('Expected CUDA int32 starts, lengths and page table')
    sequences, shape = lengths.numel(), table.shape
    if starts.numel() != sequences + 1 or len(shape) != 2 or shape[0] != sequences:
        raise ValueError('starts, lengths and page table do not match')
    stride, step = table.stride()
    if not (starts.is_contiguous() and lengths.is_contiguous()) or (step != 1 and shape[1] > 1):
        raise ValueError('starts, lengths and the rows of the page table must be contiguous')
    return (starts.data_ptr(), lengths.data_ptr(), table.data_ptr(),
            stride if sequences > 1 else shape[1], shape[1], sequences)


def check_batch(rows, k_pages, v_pages, starts, lengths, table):
    """Raises where append and paged_attention refuse these for new rows of this type and device,
    for a program that runs several operators and wants to know before the first; returns the
    cache's (kv_heads, head_dim)."""
    _, _, heads, _, dim = _cache(k_pages, v_pages, rows.dtype, rows.get_device())
    _batch(rows.get_device(), starts, lengths, table)
    return heads, dim


def append(k_pages, v_pages, k, v, starts, lengths, table, inv_freq=None, k_weight=None, q=None,
           q_weight=None, eps=1e-6):
    """Appends k and v [T, kv_heads, D] to the cache, k normed and rotated on the way
    (k_weight and inv_freq as in qk_norm_rope, by its position in its sequence).
    With q [T, q_heads, D], returns the queries normed and rotated for
    paged_attention, 0 in rows of no sequence.  The rows that a call writes must differ:
    no page twice among the new positions of its sequences."""
    k, k_token, k_head = _rows(k, 'keys')
    v, v_token, v_head = _rows(v, 'values')
    dtype, device, shape = k.dtype, k.get_device(), k.shape
    _same(v, dtype, device)
    pages, stride, heads, size, dim = _cache(k_pages, v_pages, dtype, device)
    tokens = shape[0]
    if v.shape != shape or shape[1] != heads or shape[2] != dim:
        raise ValueError('keys and values do not match the cache')
    q_args, q_out = (0, 0, 0, 0, 0, 0), None
    if q is not None:
        q, q_token, q_head = _rows(q, 'queries')
        _same(q, dtype, device)
        q_tokens, q_heads, q_dim = q.shape
        if q_tokens != tokens or q_dim != dim:
            raise ValueError('queries and keys do not match')
        q_weight, q_w = _weight(q_weight, dim, device)
        q_out = (q.new_empty if lengths.numel() else q.new_zeros)((tokens, q_heads, dim))
        q_args = (q.data_ptr(), q_token, q_head, q_heads, q_w, q_out.data_ptr())
    k_weight, k_w = _weight(k_weight, dim, device)
    inv_freq, freq, pairs = _frequencies(inv_freq, dim, device)
    _lib.launch(device, 'lm_paged_append', k.data_ptr(), k_token, k_head, k_w, v.data_ptr(),
                v_token, v_head, *q_args, k_pages.data_ptr(), v_pages.data_ptr(), pages, stride,
                heads, size, dim, *_batch(device, starts, lengths, table), freq, pairs, tokens, eps,
                _lib.dtype_code(dtype))
    return q_out


@functools.lru_cache(maxsize=1024)
def _workspace_bytes(*sizes):
    return _lib.lib().lm_paged_attention_workspace_bytes(*sizes)


def paged_attention(q, k_pages, v_pages, starts, lengths, table, scale=None, gate=None,
                    max_new=None, out=None):
    """Attention of the new tokens q [T, q_heads, D] over the cache -> [T, q_heads, D].

    The token at position p of its sequence sees the positions up to p; a row that sees none,
    or only scores of -inf, is 0.  Scores are fp32, and defined up to 2^23.  scale defaults to
    D ** -0.5; gate [T, q_heads, D] multiplies the result by sigmoid(gate).
    max_new bounds the new tokens of one sequence (default: T); a close bound saves time, and
    rows of a sequence with more may be left unwritten.  The table's width counts as a
    sequence's possible length: for one sequence of few new tokens and few keys, a wide one
    costs time and workspace (128 new tokens alone, 16 heads of 256: 39 us with 262144
    positions, 17 with 128).
    out [T, q_heads, D], contiguous, receives the result, and rows of no sequence keep what
    they hold there; without it they are 0.  It may be q or the gate itself, and shares no
    memory with them, or with the cache, in another way."""
    q, q_token, q_head = _rows(q, 'queries')
    dtype, device, shape = q.dtype, q.get_device(), q.shape
    pages, stride, heads, size, dim = _cache(k_pages, v_pages, dtype, device)
    tokens, q_heads, q_dim = shape
    if q_dim != dim or q_heads % heads:
        raise ValueError('queries do not match the cache')
    gate_args = (0, 0, 0)
    if gate is not None:
        gate, gate_token, gate_head = _rows(gate, 'gate')
        _same(gate, dtype, device)
        if gate.shape != shape:
            raise ValueError('gate does not match the queries')
        gate_args = (gate.data_ptr(), gate_token, gate_head)
    if out is None:
        out = q.new_zeros(shape)
    else:
        _same(out, dtype, device)
        if out.shape != shape or not out.is_contiguous() or out.data_ptr() % 16:
            raise ValueError('Expected a contiguous output of the shape of the queries')
    batch = _batch(device, starts, lengths, table)
    if max_new is None:
        max_new = tokens
    need = _workspace_bytes(tokens, batch[5], q_heads, heads, dim, max_new, batch[4] * size)
    workspace = q.new_empty(need // 2) if need > 0 else None
    _lib.launch(device, 'lm_paged_attention', q.data_ptr(), q_token, q_head, q_heads,
                k_pages.data_ptr(), v_pages.data_ptr(), pages, stride, heads, size, dim, *batch,
                tokens, max_new, dim ** -0.5 if scale is None else scale, *gate_args,
                out.data_ptr(), _lib.ptr(workspace), need, _lib.dtype_code(dtype))
    return out
