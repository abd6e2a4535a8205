"""Sparse self-attention module: sdd(q, k^T) -> block-sparse softmax -> dsd(p, v).

Drop-in for the reference's torch_blocksparse/deepspeedsparseselfattention.py (SparsityConfig,
DeepSpeedSparseSelfAttention); `SparseSelfAttention` is the name the same class carries in DeepSpeed.
Differences from the reference, all deliberate: the per-sequence-length operator cache is keyed by the whole
configuration instead of the sequence length alone (deepspeedsparseselfattention.py:67-106 shares operators
between modules with different layouts), and a key given as [..., head_dim, seq] is made contiguous after it is
transposed back (:119-123 hands a strided view to kernels that assume a unit inner stride).

Beyond the reference, `forward` takes score rules (`Attention`): a cap, a bias by distance, documents, a causal order with a prefix, keys and values
of fewer heads; and `decode` answers for one new position a sequence from a `KeyValueCache` over the same layout.
"""
import collections
import threading

import torch
import torch.nn as nn

from . import _lib
from .attention_core import attention_chain
from .cache import CacheAttention
from .layouts import fixed_layout
from .matmul import MatMul
from .rules import Attention
from .softmax import Softmax


class SparsityConfig:
    def __init__(self, mode='fixed', block=16, stride=64, attention='unidirectional', numverts=1, vertsize=1):
        if mode != 'dense' and mode != 'fixed':
            raise NotImplementedError('only "dense" and "fixed" modes are supported for now')
        self.mode = mode
        self.block = block
        self.stride = stride
        if attention != 'unidirectional' and attention != 'bidirectional':
            raise NotImplementedError('only "uni/bi-directional" attentions are supported for now')
        self.attention = attention
        self.numverts = numverts
        self.vertsize = vertsize

    def key(self):
        return (self.mode, self.block, self.stride, self.attention, self.numverts, self.vertsize)


class DeepSpeedSparseSelfAttention(nn.Module):

    _make_layout = staticmethod(fixed_layout)

    # Operators by (heads, sequence length, configuration, device), shared by all modules like the reference's class-level
    # cache, but bounded: the least recently used entry of a kind (the chain's, those with rules, those of decoding) goes when
    # more than OPS_CACHE_SIZE of the kind are held.
    ops = collections.OrderedDict()
    OPS_CACHE_SIZE = 16
    _lock = threading.RLock()                            # of `ops`, `captured` and `_readers`
    _readers = dict()                                    # of the chain's operators (those with rules and of decoding know their own)

    @staticmethod
    def _drop_the_oldest(key):
        """of the kind of `key`, where there are too many of it"""
        cache, kind = DeepSpeedSparseSelfAttention.ops, lambda k: k[0] if isinstance(k[0], str) else 'chain'
        alike = [k for k in cache if kind(k) == kind(key)]
        for old in alike[:-DeepSpeedSparseSelfAttention.OPS_CACHE_SIZE]:
            readers = DeepSpeedSparseSelfAttention._readers.pop(old, None)
            if readers is not None:
                readers.table(*_lib.tensors_of(cache[old]))
            del cache[old]

    def get_ops(self, H, L, device=None):
        cfg = self.sparsity_config
        key = (H, L, str(device)) + cfg.key()
        return self._held(key, lambda: self._chain(H, L, device), device)

    def _chain(self, H, L, device):
        cfg = self.sparsity_config
        num_blocks = L // cfg.block
        if num_blocks != L / cfg.block:
            raise ValueError('Sequence length %d must be dividable by block size %d' % (L, cfg.block))
        block_stride = cfg.stride // cfg.block
        if block_stride != cfg.stride / cfg.block:
            raise ValueError('Stride %d must be dividable by block size %d' % (cfg.stride, cfg.block))
        # on a GPU the layout is built there and goes straight into the table builders
        layout = DeepSpeedSparseSelfAttention._make_layout(H, num_blocks, cfg.mode, block_stride, cfg.attention,
                                                           cfg.numverts, cfg.vertsize, device=device)
        sdd_nt = MatMul(layout, cfg.block, 'sdd', trans_a=False, trans_b=True)
        dsd_nn = MatMul(layout, cfg.block, 'dsd', trans_a=False, trans_b=False)
        softmax = Softmax(layout, cfg.block)
        return sdd_nt, dsd_nn, softmax

    # Operators that a captured graph has in it: its replays use their tables, so these stay.
    captured = dict()

    @staticmethod
    def _held(key, make, device=None):
        """what `ops` holds under `key`, made where it holds nothing, for the current stream of `device`"""
        cls = DeepSpeedSparseSelfAttention
        on_gpu = isinstance(device, torch.device) and device.type == 'cuda' and device.index is not None
        with cls._lock:
            if key not in cls.ops:
                cls.ops[key] = cls.captured[key] if key in cls.captured else make()
                cls._drop_the_oldest(key)
            cls.ops.move_to_end(key)
            if (on_gpu or torch.cuda.is_available()) and torch.cuda.is_current_stream_capturing():
                cls.captured[key] = cls.ops[key]
            if on_gpu:
                readers = cls._readers.get(key)
                if readers is None:
                    readers = cls._readers[key] = _lib.Readers()
                readers.read(device)
            return cls.ops[key]

    def _kept(self, kind, H, num_blocks, make):
        """the operator `make` makes of the configuration's layout for so many blocks of any number, kept among `ops`"""
        cfg = self.sparsity_config

        def operator():
            block_stride = cfg.stride // cfg.block
            if block_stride != cfg.stride / cfg.block:
                raise ValueError('Stride %d must be dividable by block size %d' % (cfg.stride, cfg.block))
            whole = -(-num_blocks // block_stride) * block_stride        # the layout is made of whole windows
            alike = min(H, cfg.numverts)                                  # (every numverts-th head has the same one)
            layout = DeepSpeedSparseSelfAttention._make_layout(alike, whole, cfg.mode, block_stride, cfg.attention, cfg.numverts, cfg.vertsize)
            return make(layout[:, :num_blocks, :num_blocks].to(torch.uint8)[torch.arange(H, device=layout.device) % alike])

        return self._held((kind, H, num_blocks) + cfg.key(), operator)

    def __init__(self, sparsity_config=SparsityConfig(), key_padding_mask_mode='add', attn_mask_mode='mul'):
        super().__init__()
        self.sparsity_config = sparsity_config
        self.key_padding_mask_mode = key_padding_mask_mode
        self.attn_mask_mode = attn_mask_mode

    def transpose_key_for_scores(self, x, L):
        bsz, num_heads, seq_len, head_dim = x.size()
        if seq_len != L:
            return x.permute(0, 1, 3, 2).contiguous()
        return x

    def transpose_mask_for_sparse(self, qtype, x, is_key_padding_mask=False):
        x = x.type(qtype)
        if is_key_padding_mask:
            for d in range(x.dim() - 1, 0, -1):
                x = x.squeeze(dim=d)
            return x
        return x.squeeze()

    def forward(self, query, key, value, rpe=None, key_padding_mask=None, attn_mask=None, *, softcap=0., slopes=None, causal=False,
                documents=None, prefix=None):
        """Attention over the configuration's layout, scores scaled by head_dim ** -0.5.  With one of softcap, slopes, causal, documents and prefix, or with
        keys and values of fewer heads than the query, it is that of `Attention` with these rules: any length, and no rpe or masks beside them."""
        fewer_heads = query.dim() == key.dim() == 4 and key.size(1) < query.size(1)
        if softcap or slopes is not None or causal or documents is not None or prefix is not None or fewer_heads:
            if rpe is not None or key_padding_mask is not None or attn_mask is not None:
                raise ValueError('softcap, slopes, causal, documents, prefix and shared key heads do not go with rpe, key_padding_mask and attn_mask')
            if query.dim() != 4 or key.dim() != 4:
                raise ValueError('query and key must have shape [batch, heads, length, head_dim]')
            key = self.transpose_key_for_scores(key, query.size(2))
            block = self.sparsity_config.block
            op = self._kept('rules', query.size(1), -(-query.size(2) // block), lambda layout: Attention(layout, block))
            return op(query, key, value, scale=float(query.size(3)) ** -0.5, softcap=softcap, slopes=slopes, causal=causal, documents=documents, prefix=prefix)
        bsz, num_heads, tgt_len, head_dim = query.size()
        key = self.transpose_key_for_scores(key, tgt_len)
        if query.shape != key.shape or key.shape != value.shape:
            raise NotImplementedError('only self-attention is supported for now')
        if key_padding_mask is not None:
            key_padding_mask = self.transpose_mask_for_sparse(query.dtype, key_padding_mask, is_key_padding_mask=True)
        if attn_mask is not None:
            attn_mask = self.transpose_mask_for_sparse(query.dtype, attn_mask)
        sdd_nt, dsd_nn, softmax = self.get_ops(num_heads, tgt_len, query.device)
        scaling = float(head_dim) ** -0.5
        # the reference's three calls (deepspeedsparseselfattention.py:152-157), in one launch where the kernels allow it
        return attention_chain(sdd_nt, softmax, dsd_nn, query, key, value, scale=scaling, rpe=rpe,
                               key_padding_mask=key_padding_mask, attn_mask=attn_mask,
                               key_padding_mask_mode=self.key_padding_mask_mode, attn_mask_mode=self.attn_mask_mode)

    def decode(self, query, cache, table, lengths, *, softcap=0., slopes=None):
        """One new position a sequence: query [batch, heads, head_dim] over the pages `table` [batch, width] of `cache`, which hold `lengths` [batch]
        positions of each sequence, the new one among them (`CacheAttention`).  It is what `forward` with causal=True and the same softcap and slopes gives
        for each sequence's last position, over keys and values as the cache holds them."""
        if query.dim() != 3 or table.dim() != 2:
            raise ValueError('query must have shape [batch, heads, head_dim], table [batch, width]')
        cfg = self.sparsity_config
        # Rows of the layout are the same in a longer one, as far as a position sees: one operator serves a quarter of an octave of widths, and a
        # table that grows by a page finds it made.  Where everything is seen no layout is needed.
        if cfg.mode == 'dense':
            blocks, make = 0, lambda layout: CacheAttention(cfg.block)
        else:
            unit = max(16, 1 << max(0, table.size(1).bit_length() - 3))
            blocks, make = -(-max(1, table.size(1)) // unit) * unit, lambda layout: CacheAttention(cfg.block, layout)
            if blocks > 65535 >= table.size(1):
                blocks = 65535                           # (the longest that CacheAttention takes)
        op = self._kept('decode', query.size(1), blocks, make)
        return op(query, cache, table, lengths, scale=float(query.size(2)) ** -0.5, softcap=softcap, slopes=slopes)


SparseSelfAttention = DeepSpeedSparseSelfAttention
