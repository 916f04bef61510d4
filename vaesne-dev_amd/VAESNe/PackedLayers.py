"""Layers of a transformer over packed sequences: batches whose sequences have different lengths lie
one behind the other, without padding, in fp32, bf16 or fp16.

    seqs = PackedSequences([37, 60, 21])                   # once per batch
    x = torch.cat(light_curves)                            # [118, model_dim]
    block = PackedTransformerBlock(model_dim, heads, ff_dim, buckets=RelativeBuckets(32, 128))
    x, n = block(x, block.enter(x), seqs)                  # -> the residual stream and its norm

The operators stand by themselves too: packed_attention, gated_norm, pre_norm, gelu8, linear8, pack8,
unpack8.  The padded layers of util_layers (fp32, key padding masks, dropout) are unchanged;
PackedSequences.from_mask takes one of their batches over.  Every call is a launch of a hand-written
gfx950 kernel (include/vaesne_hip.h), but for the plain products of Linear layers; there is no CPU path.
Derivatives are first-order and reverse-mode: a second one raises, and so does a tensor with a forward-mode tangent.
"""
from __future__ import annotations

import torch
from torch import nn

from . import _packed_ops
from ._packed_ops import Packed8, PackedSequences, RelativeBuckets, pack8, unpack8

__all__ = ["PackedSequences", "RelativeBuckets", "Packed8", "packed_attention", "gated_norm", "pre_norm", "gelu8",
           "linear8", "pack8", "unpack8", "RelativeBias", "GatedNorm", "PackedTransformerBlock"]


def packed_attention(q, k, v, seqs, causal=False, scale=None, bias=None, buckets=None):
    """Softmax attention over packed sequences -> [queries, heads, dim].

    q [queries, heads, dim]; k, v [keys, key heads, dim], the heads a multiple of the key heads (each
    key head serves heads / key heads neighbouring ones); dim a multiple of 8 up to 128.  Slices of a
    wider tensor (a q | k | v product) are read in place where their rows are 16-byte aligned.

    seqs: the PackedSequences of q and k.  A sequence's queries are the last positions of its keys,
    so with `causal` query i sees keys 0 .. i + (keys - queries); a query that sees none
    gives zeros and no gradient.  scale: default dim ** -0.5.  bias [buckets, heads] with `buckets`
    (RelativeBuckets): bias[bucket(key position - query position), head] is added to the scaled score; one below
    -11356, as -inf, masks its keys.
    Gradients for q, k, v and bias; results are bitwise reproducible.  Sums and softmax statistics are fp32; in
    16-bit types the probabilities and (in the backward pass) their gradients are rounded to the type before their products
    on the matrix cores, fp16's gradients in two parts, and rowsum(dout * out) takes the rounded output (bf16's bias
    gradient: the probabilities).  An infinity or NaN reaches queries and keys of its own sequence only (with `causal`,
    also earlier ones in it).  No dropout."""
    return _packed_ops.packed_attention(q, k, v, seqs, causal, scale, bias, buckets)


def gated_norm(x, branch, pre_weight, post_weight, pre_bias=None, post_bias=None, gate=None, residual_scale=1.0,
               kind="rms", eps=1e-5):
    """The join between two blocks in one pass -> (y, n):

        y = residual_scale * x + gate * N(branch; post_weight, post_bias)
        n = N(y; pre_weight, pre_bias)

    x the residual stream [..., channels] (at most 8192), branch the block's output; N over the last
    axis, kind "rms" or "layer" (with optional biases).  gate: None, one value per channel, or one per
    token and channel.  n is taken from y before y is rounded to the tensors' type.  Gradients for
    every tensor."""
    return _packed_ops.gated_norm(x, branch, pre_weight, post_weight, pre_bias, post_bias, gate, residual_scale, kind,
                                  eps)


def pre_norm(x, weight, bias=None, kind="rms", eps=1e-5):
    """The norm before a first block: gated_norm's n without a branch."""
    return _packed_ops.pre_norm(x, weight, bias, kind, eps)


def gelu8(x):
    """GELU(x) (erf form) that keeps x for its backward pass in 8 bits (pack8's form): the output is that of
    the exact x, the gradient is dy * GELU'(kept x).  Errors are relative to the result, far into the negative
    tail: the rounding to the type and a 30th of it more (fp32: 8 of 2^-24 in all); below 2^-126 it is 0."""
    return _packed_ops.gelu8(x)


def linear8(x, weight, bias=None, act=None):
    """act(x) weight^T + bias, act None or "gelu", with x kept for the backward pass in 8 bits: the
    output is that of the exact x, the weight's gradient takes act(kept x).  Inside autocast too the result has
    the tensors' own type."""
    return _packed_ops.linear8(x, weight, bias, act)


class RelativeBias(nn.Module):
    """A learned bias for each bucket of relative positions and head: weight [buckets, heads], zeros at
    first."""

    def __init__(self, buckets, num_heads):
        super().__init__()
        self.buckets = buckets
        self.weight = nn.Parameter(torch.zeros(buckets.num_buckets, num_heads))


class GatedNorm(nn.Module):
    """gated_norm with its parameters: weights 1, biases 0, a gate per channel of `gate` (None: none)."""

    def __init__(self, channels, kind="rms", gate=None, residual_scale=1.0, eps=1e-5):
        super().__init__()
        if kind not in _packed_ops.KINDS:
            raise ValueError("GatedNorm: kind is 'rms' or 'layer'")
        self.kind, self.residual_scale, self.eps = kind, residual_scale, eps
        self.pre_weight = nn.Parameter(torch.ones(channels))
        self.post_weight = nn.Parameter(torch.ones(channels))
        layer = kind == "layer"
        self.pre_bias = nn.Parameter(torch.zeros(channels)) if layer else None
        self.post_bias = nn.Parameter(torch.zeros(channels)) if layer else None
        self.gate = None if gate is None else nn.Parameter(torch.full((channels,), float(gate)))

    def forward(self, x, branch, gate=None):
        """(y, n); `gate` [.., channels]: per token, in place of the module's own."""
        return gated_norm(x, branch, self.pre_weight, self.post_weight, self.pre_bias, self.post_bias,
                          self.gate if gate is None else gate, self.residual_scale, self.kind, self.eps)


class PackedTransformerBlock(nn.Module):
    """Self-attention and a GELU feed-forward over packed sequences, each followed by its gated norm
    join, feed-forward activations kept in 8 bits:

        a = out(attention(qkv(n)));  x, n = join1(x, a);  f = W2 gelu(W1 n);  x, n = join2(x, f)

    The block takes the residual stream x and its norm n and returns the next pair: one pass over the tokens
    between out's product and the feed-forward, and between two blocks.  `enter` is the norm before the first block."""

    def __init__(self, embed_dim, num_heads, ff_dim, num_kv_heads=None, causal=False, buckets=None, kind="rms",
                 gate=None, residual_scale=1.0):
        super().__init__()
        num_kv_heads = num_heads if num_kv_heads is None else num_kv_heads
        if embed_dim % num_heads or num_heads % num_kv_heads:
            raise ValueError("PackedTransformerBlock: embed_dim / num_heads and num_heads / num_kv_heads are whole numbers")
        self.num_heads, self.num_kv_heads, self.head_dim = num_heads, num_kv_heads, embed_dim // num_heads
        self.causal = causal
        self.enter_weight = nn.Parameter(torch.ones(embed_dim))
        self.kind = kind
        self.qkv = nn.Linear(embed_dim, (num_heads + 2 * num_kv_heads) * self.head_dim)
        self.out = nn.Linear(embed_dim, embed_dim)
        self.up = nn.Linear(embed_dim, ff_dim)
        self.down = nn.Linear(ff_dim, embed_dim)
        self.relative = None if buckets is None else RelativeBias(buckets, num_heads)
        self.join1 = GatedNorm(embed_dim, kind, gate, residual_scale)
        self.join2 = GatedNorm(embed_dim, kind, gate, residual_scale)

    def enter(self, x):
        return pre_norm(x, self.enter_weight, kind=self.kind)

    def forward(self, x, n, seqs):
        H, Hk, D = self.num_heads, self.num_kv_heads, self.head_dim
        q, k, v = self.qkv(n).view(-1, H + 2 * Hk, D).split([H, Hk, Hk], 1)
        more = {} if self.relative is None else {"bias": self.relative.weight, "buckets": self.relative.buckets}
        a = packed_attention(q, k, v, seqs, causal=self.causal, **more)
        x, n = self.join1(x, self.out(a.reshape(-1, H * D)))
        h = linear8(n, self.up.weight, self.up.bias)
        return self.join2(x, linear8(h, self.down.weight, self.down.bias, act="gelu"))
