"""The attention half of a decoder layer over a paged cache, as MoEStack runs it before a
layer's MoE block:

  h += o( attention( rotate(norm(q)), cache ) * sigmoid(gate) ),  [q, gate, k, v] = qkv(rmsnorm(h))

with int8 projections (operators/int8.linear), the norms, rotation and append in one launch
and paged attention (operators/attention).  Rows, heads and weights are laid out as the
Transformers module has them (HF:627-735): a head's query and gate side by side, norm
weights as 1 + w, the first channels of a head rotated in two halves.  The reference runs
the Transformers module itself; its cache is a contiguous one per request
(generation.py:32).
"""
from typing import NamedTuple

import torch

from .. import router
from ..operators import attention, int8


class Batch(NamedTuple):
    """What a step's attention works on, the same for every layer: starts [sequences + 1],
    lengths [sequences] and page table [sequences, n], int32 on the GPU (operators/attention),
    and the most new tokens of a sequence (None: not known)."""
    starts: torch.Tensor
    lengths: torch.Tensor
    table: torch.Tensor
    max_new: int | None = None


class AttentionBlock:
    """One layer's attention: weights, norms and its pages.

    qkv and o are {'q': int8 [N, K], 'scale': fp32 [N, K / 128]} as quantize_g128 and
    Artifact.quantized give them; the rows of qkv are each head's query and, if gated, its
    gate, then the keys, then the values.  norm [H], q_norm and k_norm [head_dim] are RMSNorm
    weights w of (1 + w), None for zeros (norm) or no norm (q_norm, k_norm)."""

    def __init__(self, qkv, o, q_heads, kv_heads, head_dim, norm=None, q_norm=None, k_norm=None,
                 inv_freq=None, gated=True, eps=1e-6):
        self.qkv, self.o = qkv, o
        self.q_heads, self.kv_heads, self.head_dim = q_heads, kv_heads, head_dim
        self.norm, self.q_norm, self.k_norm = norm, q_norm, k_norm
        self.inv_freq, self.gated, self.eps = inv_freq, gated, eps
        self.q_width = q_heads * head_dim * (2 if gated else 1)
        self.kv_width = kv_heads * head_dim
        if (qkv['q'].shape[0] != self.q_width + 2 * self.kv_width
                or o['q'].shape[1] != q_heads * head_dim or o['q'].shape[0] != qkv['q'].shape[1]):
            raise ValueError('the projections do not match the heads')
        # what the operators would refuse in every step
        if head_dim not in (64, 128, 256) or min(q_heads, kv_heads) < 1 or q_heads % kv_heads:
            raise ValueError('expected heads of 64, 128 or 256, and query heads a multiple of '
                             'key-value heads')
        for bank in (qkv, o):
            if bank['q'].shape[1] % 128:
                raise ValueError('projections have groups of 128')
            if tuple(bank['scale'].shape) != (bank['q'].shape[0], bank['q'].shape[1] // 128):
                raise ValueError('the scales do not match their projection')
        for w, n in ((norm, qkv['q'].shape[1]), (q_norm, head_dim), (k_norm, head_dim)):
            if w is not None and w.numel() != n:
                raise ValueError('norm weight does not match its rows')
        attention.check_frequencies(inv_freq, head_dim)
        self.k_pages = self.v_pages = None

    def allocate(self, pages, page_size=64, dtype=torch.bfloat16):
        """An empty cache of `pages` pages for this layer, of bf16 like the rows that forward_
        takes."""
        if dtype is not torch.bfloat16:
            raise ValueError('the block appends bf16 keys and values')
        if not 16 <= page_size <= 1024 or page_size & (page_size - 1):
            raise ValueError('page size must be a power of two from 16 to 1024')
        shape = (pages, self.kv_heads, page_size, self.head_dim)
        device = self.qkv['q'].device
        self.k_pages = torch.empty(shape, dtype=dtype, device=device)
        self.v_pages = torch.empty(shape, dtype=dtype, device=device)
        return self

    def check(self, h, batch):
        """Raises for rows h, a batch and a cache that forward_ refuses."""
        self._check_rows(h, batch)
        if (not h.is_cuda or h.dtype is not torch.bfloat16
                or h.shape[1] != self.qkv['q'].shape[1]):
            raise ValueError('expected CUDA bf16 rows [tokens, hidden]')
        shape = attention.check_batch(h, self.k_pages, self.v_pages, batch.starts, batch.lengths,
                                      batch.table)
        if shape != (self.kv_heads, self.head_dim):
            raise ValueError('the pages do not match the heads')

    def _check_rows(self, h, batch):
        """Of that, what the operators before the append would not find."""
        if self.k_pages is None:
            raise RuntimeError('allocate() the pages of the attention layers first')
        if h.ndim != 2:
            raise ValueError('expected rows [tokens, hidden]')
        if batch.max_new is not None and batch.max_new < 0:
            raise ValueError('invalid number of new tokens')

    def forward_(self, h, batch):
        """h [T, H] bf16, updated in place: h += block(h); the new tokens' keys and values join
        the cache.  Rows of no sequence stay as they are.  Nothing is written before a call is
        refused."""
        self._check_rows(h, batch)
        tokens, dim = h.shape[0], self.head_dim
        x = int8.linear(router.rmsnorm(h, self.norm, self.eps), self.qkv['q'], self.qkv['scale'])
        q, k, v = x.split([self.q_width, self.kv_width, self.kv_width], dim=1)
        q, gate = q.view(tokens, self.q_heads, self.q_width // self.q_heads), None
        if self.gated:
            q, gate = q[..., :dim], q[..., dim:]
        k, v = (t.view(tokens, self.kv_heads, dim) for t in (k, v))
        place = batch.starts, batch.lengths, batch.table
        q = attention.append(self.k_pages, self.v_pages, k, v, *place, inv_freq=self.inv_freq,
                             k_weight=self.k_norm, q=q, q_weight=self.q_norm, eps=self.eps)
        o = attention.paged_attention(q, self.k_pages, self.v_pages, *place, gate=gate,
                                      max_new=batch.max_new)
        h += int8.linear(o.view(tokens, self.q_heads * dim), self.o['q'], self.o['scale'])
        return h
