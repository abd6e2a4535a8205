"""Block-sparse attention whose scores follow rules: a cap, a bias by distance, documents, a causal order with a prefix.

`Attention(layout, block)(q, k, v, ...)` is the chain scores -> softmax -> context of the attention modules for models whose masks
and biases are functions of the positions.  The modules take those as tensors of every pair (`rpe`, `attn_mask`); here they are a few
numbers per row or head and no pair of positions costs memory:

    y_ij = softcap * tanh(scale * q_i . k_j / softcap) - slopes[h] * |i - j|        (softcap 0: scale * q_i . k_j - ...)
    o_i  = sum_j softmax_j(y_ij) v_j   over the keys j that row i sees

Row i sees key j if block (h, i // block, j // block) is in the layout, if documents[z, i] == documents[z, j] >= 0 (where documents
are given) and, with causal, if j <= i or j < prefix[z].  A row that sees no key gets zeros, as result and as gradient.  Positions
with a negative document number (padding) see nothing and are seen by nothing: what q, k, v and the incoming gradient hold there
reaches no result, NaN included.  At positions that some rows see, a NaN or an infinity in v (in the backward pass, in any operand) can make
rows NaN that do not see it, as 0 * NaN does in a product with a masked softmax.

Sums, statistics and score gradients' factors are fp32; shares and score gradients are rounded to the operands' type where they become an operand of a
product (16-bit types: those of the gradient of q in two terms, with `shared` all of them).  In float16 the backward pass's shares, which are normalised, and score gradients lose bits where they are below 2^-14, as every share of a row of more than some
16000 equal keys is.  With a backward pass to follow a 16-bit call keeps, beside its operands and result, a tensor as large as the result (what its rounding left out).

One kernel forward, two backward (rows: dq; columns: dk and dv), none of which stores a sparse tensor (bsp_attention_rules_fwd,
bsp_attention_rules_bwd).  The results of a call are the same bits every time.
"""
import ctypes
import struct

import torch
from torch.autograd.function import once_differentiable

from . import _lib


# bsp_attention_rules_call: dtype, Z, H, kv_heads, lines, D; length, strides[24]; scale, softcap, causal; slopes, documents, documents_stride, prefix, ranges, d_rows, stats, o_rest
_CALL = struct.Struct('@6i25q2fiPPqPPPPP')


def _operand(t, Z, heads, L, D):
    """(t, or a copy of it where the kernels could not address t: unit inner stride, 16-byte vectors, rows that do not overlap and lie within 4 GiB of a
    head's first; its batch, head and row stride, those that no address depends on as the kernels want them)"""
    z, h, row, one = t.stride()
    z, h, row = z if Z > 1 else 0, h if heads > 1 else 0, row if L > 1 else D
    size = t.element_size()
    if one == 1 and not (z | h | row) * size % 16 and row >= D and not t.data_ptr() % 16 and row * (L + 64) * size < 1 << 32:
        return t, (z, h, row)
    return t.clone(memory_format=torch.contiguous_format), _own(Z, heads, L, D)


def _own(Z, heads, L, D):
    """the strides of a contiguous tensor"""
    return (heads * L * D if Z > 1 else 0, L * D if heads > 1 else 0, D)


def check_scores(scale, softcap):
    """a capped score is off by softcap * 2^-23 (the tanh comes of an exponential in fp32), so a cap has an upper end"""
    if not (softcap == 0. or 2. ** -10 <= softcap <= 1024.):
        raise ValueError('softcap must be 0 or between 2^-10 and 1024 (got %s)' % softcap)
    if not abs(scale) <= 2. ** 100:
        raise ValueError('scale must be finite, 2^100 at most (got %s)' % scale)


def _at(t):
    return 0 if t is None else t.data_ptr()


MOST_PLACES = 2 ** 31 - 1     # places in a table are 32-bit numbers


def _places(n):
    if n > MOST_PLACES:
        raise ValueError('the tables of the layout take %d numbers, more than %d' % (n, MOST_PLACES))


class _Tables:
    """The tables of a layout on one device: the lines of 64 rows, and per number of query heads that share a key head the columns of
    64 keys (bsp_attention_tables_build)."""

    def __init__(self, layout, block, device):
        lay = (layout != 0).cpu()
        if block > 64:                     # larger blocks are read as blocks of 64
            lay = lay.repeat_interleave(block // 64, 1).repeat_interleave(block // 64, 2)
        self.block, self.device = min(block, 64), device
        S = 64 // self.block
        self.layout = torch.nn.functional.pad(lay.to(torch.uint8), (0, -lay.size(2) % S, 0, -lay.size(1) % S)).contiguous()
        host, info = self._build(self.layout)
        _places(info.items_offset)
        self.lines = info.lines
        self.rows = host[:info.items_offset].to(device)
        self._columns, self._chosen = dict(), dict()
        self.readers = _lib.Readers()
        self.readers.table(self.rows)

    def _build(self, lay):
        H, R, C = lay.shape
        info = _lib.AttentionTables()
        cap = 32 * H * (R + C) + 16 * int(torch.count_nonzero(lay)) + 64
        host = torch.empty(cap, dtype=torch.int32, device='cpu')
        _lib.check(_lib.load().bsp_attention_tables_build(_lib.ptr(lay), H, R, C, self.block, _lib.ptr(host), cap, ctypes.byref(info)), 'bsp_attention_tables_build')
        return host, info

    # Work items of the columns for a launch over `batches` sequences: a column of many tiles is cut into parts, so that the longest do not
    # outlast the launch (twice the average, as in the tables of the other kernels, or half of what each of some WANTED workgroups at a time
    # has to do: the longest go first) and a small launch still has some WANTED items for its 256 compute units; every part costs a slot of 512 D bytes
    # written and read (fp16 8 x 16 x 4096, blocks of 16, stride 64: parts of 21, 32 and 64 tiles 334, 322 and 329 us).
    WANTED = 1024

    def columns(self, kv_heads, batches):
        """(items, their number per key head, splits, number of splits, slots), tensors on the device"""
        made = self._chosen.get((kv_heads, batches))
        if made is None:
            made = self._chosen[kv_heads, batches] = self._choose(kv_heads, batches)
        return made

    def _choose(self, kv_heads, batches):
        H, R, C = self.layout.shape
        tiles = self._columns.get(kv_heads)
        if tiles is None:
            host, info = self._build(self.layout.view(kv_heads, H // kv_heads * R, C))
            items = host[info.items_offset:info.split_offset]
            heads = items[:12 * info.n_items].view(-1, 12).clone()
            begin = -(-12 * info.n_items // 8) * 8                   # (entries start at a multiple of eight ints)
            entries = items[begin:].view(-1, 8).clone()
            if kv_heads != H:              # positions of the stacked query heads -> query head and position in it
                length = R * self.block
                entries[:, :4] = (entries[:, :4] // length << 24) + entries[:, :4] % length
            # the builder's own parts of a column are joined again: by key head and column, in the order of their entries
            column = heads[:, 2].long() * info.columns + heads[:, 3]
            order = torch.argsort(column * (len(entries) + 1) + (heads[:, 1] - begin) // 8)
            heads, column = heads[order], column[order]
            first = (heads[:, 1].long() - begin) // 8
            whole = torch.ones(info.n_items, dtype=torch.bool, device='cpu')
            whole[1:] = column[1:] != column[:-1]
            group = whole.cumsum(0) - 1
            count = torch.zeros(int(group[-1]) + 1, dtype=torch.long, device='cpu').index_add_(0, group, heads[:, 0].long())
            tiles = self._columns[kv_heads] = (heads[whole], first[whole], count, entries, dict())
        heads, first, count, entries, made = tiles
        total, n = int(count.sum()), count.numel()
        part = max(16, min(max(-(-2 * total // n), batches * total // (2 * self.WANTED) // 16 * 16), int(count.max())))    # (few different ones: each is a table that is kept)
        while part > 4 and batches * int(((count + part - 1) // part).clamp(min=1).sum()) < self.WANTED:
            part //= 2
        if part not in made:
            made[part] = self._cut(heads, first, count, entries, part)
            self.readers.table(made[part][0], made[part][2])
        return made[part]

    def _cut(self, heads, first, count, entries, part):
        parts = ((count + part - 1) // part).clamp(min=1)
        of = torch.repeat_interleave(torch.arange(count.numel(), device='cpu'), parts)
        k = torch.arange(of.numel(), device='cpu') - (parts.cumsum(0) - parts)[of]
        base, rest = (count // parts)[of], (count % parts)[of]
        items = heads[of].clone()
        items[:, 0] = (base + (k < rest)).int()
        items[:, 1] = (8 * (first[of] + k * base + torch.minimum(k, rest))).int()
        split = parts[of] > 1
        items[:, 4] = torch.where(split, split.long().cumsum(0) - 1, -1).int()
        slots = int(split.sum())
        cut = parts > 1
        splits = torch.stack([heads[cut, 2], heads[cut, 3], (parts[cut].cumsum(0) - parts[cut]).int(), parts[cut].int()] + [heads[cut, 8 + g] for g in range(4)], 1)
        # by key head, the longest first, every key head's list filled up to the longest of them
        kv_heads = int(heads[:, 2].max()) + 1
        order = torch.argsort(items[:, 2].long() * (1 << 32) - items[:, 0], stable=True)
        items, number = items[order], torch.bincount(items[:, 2].long(), minlength=kv_heads)
        n_items = int(number.max())
        rank = torch.arange(of.numel(), device='cpu') - (number.cumsum(0) - number)[items[:, 2].long()]
        begin = 12 * kv_heads * n_items
        _places(begin + entries.numel())
        lists = torch.zeros((kv_heads, n_items, 12), dtype=torch.int32, device='cpu')
        lists[:, :, 1], lists[:, :, 3], lists[:, :, 4] = begin, -1, -1
        lists[items[:, 2].long(), rank] = items
        lists[:, :, 1] += begin * (lists[:, :, 3] >= 0)
        dev = torch.cat([lists.flatten(), entries.flatten()]).to(self.device)
        return dev, n_items, splits.contiguous().to(self.device) if slots else None, splits.size(0), slots


class _rules(torch.autograd.Function):

    @staticmethod
    def forward(ctx, q, k, v, tables, scale, softcap, slopes, causal, documents, prefix, grad_enabled):
        Z, H, L, D = q.shape
        kv, device = k.size(1), q.device
        (q, q_at), (k, k_at), (v, v_at) = _operand(q, Z, H, L, D), _operand(k, Z, kv, L, D), _operand(v, Z, kv, L, D)
        keep = grad_enabled and any(ctx.needs_input_grad[:3])
        o = torch.empty_like(q, memory_format=torch.contiguous_format)
        stats = torch.empty((Z, H, 2, 64 * tables.lines), dtype=torch.float32, device=device) if keep else None
        rest = torch.empty_like(q, memory_format=torch.contiguous_format) if keep and q.element_size() == 2 else None
        ranges = torch.empty((Z, (L + 15) // 16, 2), dtype=torch.int32, device=device) if documents is not None else None
        call = _rules.call(q, kv, q_at + k_at + v_at + _own(Z, H, L, D) + (0,) * 12, tables, scale, softcap, slopes, causal, documents, prefix, ranges, stats, rest)
        rc = _lib.load().bsp_attention_rules_fwd(call, q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), _lib.raw_stream(device))
        if rc:
            _lib.check(rc, 'bsp_attention_rules_fwd')
        if keep:
            ctx.save_for_backward(q, k, v, o, rest, stats, ranges, slopes, documents, prefix)
            ctx.tables, ctx.numbers = tables, (scale, softcap, causal)
        return o

    @staticmethod
    def call(q, kv, strides, tables, scale, softcap, slopes, causal, documents, prefix, ranges, stats, rest):
        Z, H, L, D = q.shape
        return _CALL.pack(_lib.DTYPES[q.dtype], Z, H, kv, tables.lines, D, L, *strides, scale, softcap, causal, _at(slopes), _at(documents),
                          documents.stride(0) if documents is not None and Z > 1 else 0, _at(prefix), _at(ranges), tables.rows.data_ptr(), _at(stats), _at(rest))

    @staticmethod
    @once_differentiable
    def backward(ctx, do):
        q, k, v, o, rest, stats, ranges, slopes, documents, prefix = ctx.saved_tensors
        tables, (scale, softcap, causal) = ctx.tables, ctx.numbers
        need_q, need_k, need_v = ctx.needs_input_grad[:3]
        device, dtype = q.device, q.dtype
        with _lib.on_device(device):
            Z, H, L, D = q.shape
            kv = k.size(1)
            # (what was saved may have been elsewhere in between and have come back in other strides)
            (q, q_at), (k, k_at), (v, v_at) = _operand(q, Z, H, L, D), _operand(k, Z, kv, L, D), _operand(v, Z, kv, L, D)
            (o, o_at), (do, do_at) = _operand(o, Z, H, L, D), _operand(do, Z, H, L, D)
            dq, dk, dv = torch.empty_like(q, memory_format=torch.contiguous_format), None, None
            delta = torch.empty((Z, H, 64 * tables.lines), dtype=torch.float32, device=device)
            items, n_items, splits, n_splits, slots, partial = None, 0, None, 0, 0, None
            if need_k or need_v:
                dk, dv = [torch.empty_like(t, memory_format=torch.contiguous_format) for t in (k, v)]
                items, n_items, splits, n_splits, slots = tables.columns(kv, Z)
                partial = torch.empty((Z, slots, 2, 64, D), dtype=torch.float32, device=device) if slots else None
            own = _own(Z, kv, L, D)
            call = _rules.call(q, kv, q_at + k_at + v_at + o_at + do_at + _own(Z, H, L, D) + own + own, tables, scale, softcap, slopes, causal, documents, prefix, ranges, stats, rest)
            rc = _lib.load().bsp_attention_rules_bwd(call, do.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), dq.data_ptr(), _at(dk), _at(dv), delta.data_ptr(),
                                                     _at(items), n_items, _at(partial), slots, _at(splits), n_splits, _lib.raw_stream(device))
            if rc:
                _lib.check(rc, 'bsp_attention_rules_bwd')
        return dq if need_q else None, dk if need_k else None, dv if need_v else None, None, None, None, None, None, None, None, None


# bsp_attention_shared_part: q, k; strides[10]; dq, dk, dk_heads
_PART = struct.Struct('@2P10q3P')
SHARED = 64                   # elements of a key part that all heads share


class _shared_rules(torch.autograd.Function):
    """_rules with a part q_s [Z, H, L, 64] . k_s [Z, L, 64] of the scores, k_s for all heads"""

    @staticmethod
    def _parts(q_s, k_s):
        Z, H, L, _ = q_s.shape
        (q_s, q_at), (k_s, k_at) = _operand(q_s, Z, H, L, SHARED), _operand(k_s.unsqueeze(1), Z, 1, L, SHARED)
        return q_s, q_at, k_s, (k_at[0], k_at[2])

    @staticmethod
    def forward(ctx, q, k, v, q_s, k_s, tables, scale, softcap, slopes, causal, documents, prefix, grad_enabled):
        Z, H, L, D = q.shape
        kv, device = k.size(1), q.device
        (q, q_at), (k, k_at), (v, v_at) = _operand(q, Z, H, L, D), _operand(k, Z, kv, L, D), _operand(v, Z, kv, L, D)
        own_k_s = k_s
        q_s, qs_at, k_s, ks_at = _shared_rules._parts(q_s, k_s)
        keep = grad_enabled and any(ctx.needs_input_grad[:5])
        o = torch.empty_like(q, memory_format=torch.contiguous_format)
        stats = torch.empty((Z, H, 2, 64 * tables.lines), dtype=torch.float32, device=device) if keep else None
        rest = torch.empty_like(q, memory_format=torch.contiguous_format) if keep and q.element_size() == 2 else None
        ranges = torch.empty((Z, (L + 15) // 16, 2), dtype=torch.int32, device=device) if documents is not None else None
        call = _rules.call(q, kv, q_at + k_at + v_at + _own(Z, H, L, D) + (0,) * 12, tables, scale, softcap, slopes, causal, documents, prefix, ranges, stats, rest)
        part = _PART.pack(q_s.data_ptr(), k_s.data_ptr(), *qs_at, *ks_at, 0, 0, 0, 0, 0, 0, 0, 0)
        rc = _lib.load().bsp_attention_shared_fwd(call, part, q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), _lib.raw_stream(device))
        if rc:
            _lib.check(rc, 'bsp_attention_shared_fwd')
        if keep:
            ctx.save_for_backward(q, k, v, q_s, own_k_s, o, rest, stats, ranges, slopes, documents, prefix)
            ctx.tables, ctx.numbers = tables, (scale, softcap, causal)
        return o

    @staticmethod
    @once_differentiable
    def backward(ctx, do):
        q, k, v, q_s, k_s, o, rest, stats, ranges, slopes, documents, prefix = ctx.saved_tensors
        tables, (scale, softcap, causal) = ctx.tables, ctx.numbers
        need = ctx.needs_input_grad[:5]
        device, dtype = q.device, q.dtype
        with _lib.on_device(device):
            Z, H, L, D = q.shape
            kv = k.size(1)
            (q, q_at), (k, k_at), (v, v_at) = _operand(q, Z, H, L, D), _operand(k, Z, kv, L, D), _operand(v, Z, kv, L, D)
            (o, o_at), (do, do_at) = _operand(o, Z, H, L, D), _operand(do, Z, H, L, D)
            q_s, qs_at, k_s, ks_at = _shared_rules._parts(q_s, k_s)
            dq, dq_s = [torch.empty_like(t, memory_format=torch.contiguous_format) for t in (q, q_s)]
            dk = dv = dk_s = heads = None
            delta = torch.empty((Z, H, 64 * tables.lines), dtype=torch.float32, device=device)
            items, n_items, splits, n_splits, slots, partial = None, 0, None, 0, 0, None
            if need[1] or need[2] or need[4]:
                dk, dv = [torch.empty_like(t, memory_format=torch.contiguous_format) for t in (k, v)]
                dk_s, heads = torch.empty((Z, L, SHARED), dtype=dtype, device=device), torch.empty((Z, kv, L, SHARED), dtype=torch.float32, device=device)
                items, n_items, splits, n_splits, slots = tables.columns(kv, Z)
                partial = torch.empty((Z, slots, 64, 2 * D + SHARED), dtype=torch.float32, device=device) if slots else None
            own = _own(Z, kv, L, D)
            call = _rules.call(q, kv, q_at + k_at + v_at + o_at + do_at + _own(Z, H, L, D) + own + own, tables, scale, softcap, slopes, causal, documents, prefix, ranges, stats, rest)
            part = _PART.pack(q_s.data_ptr(), k_s.data_ptr(), *qs_at, *ks_at, *_own(Z, H, L, SHARED), L * SHARED, SHARED, dq_s.data_ptr(), _at(dk_s), _at(heads))
            rc = _lib.load().bsp_attention_shared_bwd(call, part, do.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), dq.data_ptr(), _at(dk), _at(dv), delta.data_ptr(),
                                                      _at(items), n_items, _at(partial), slots, _at(splits), n_splits, _lib.raw_stream(device))
            if rc:
                _lib.check(rc, 'bsp_attention_shared_bwd')
        return tuple(g if n else None for g, n in zip((dq, dk, dv, dq_s, dk_s), need)) + (None,) * 8


class Attention:
    """Attention over a block-sparse layout [heads, blocks, blocks] (block 16, 32, 64 or 128) with score rules.

    Called with q [batch, heads, length, dim] and k, v [batch, key heads, length, dim]: dim 64 or 128, float16, bfloat16 or float32, the
    number of heads a multiple of that of the key heads (query head h uses key head h // (heads / key heads)), any length that ends in the
    layout's last block.

    scale     factor of the scores
    softcap   0 for none, else the scores are softcap * tanh(scale * q . k / softcap); 2^-10 to 1024
    slopes    None, or [heads] float32: slopes[h] * |i - j| is taken off the scores (constants: refused where they require a gradient, but under no_grad)
    causal    row i sees the keys up to i only
    documents None, or [batch, length] int32: a row sees keys of its own document only; negative: padding
    prefix    None, or [batch] int32, with causal: keys before prefix[z] are seen by every row
    shared    None, or (q_s [batch, heads, length, 64], k_s [batch, length, 64]): scale * (q . k + q_s . k_s) in the place of scale * q . k, with one k_s for all heads, as latent attention
              has where its keys and values are expanded (`LatentAttention` is its other form)

    Differentiable in q, k, v and shared, once.  Tables are made at the first call on a device (for a backward pass, at the first
    one), so a call that is captured into a graph needs one like it before."""

    def __init__(self, layout, block):
        if layout.dim() != 3 or layout.size(1) != layout.size(2):
            raise ValueError('layout must have shape [heads, blocks, blocks]')
        if block not in (16, 32, 64, 128):
            raise ValueError('block must be 16, 32, 64 or 128 (got %s)' % (block,))
        if layout.size(0) > 0 and layout.size(1) * block >= 1 << 24:
            raise ValueError('the layout covers %d positions, more than 2^24' % (layout.size(1) * block))
        self.layout, self.block = layout, block
        self._tables = dict()

    def tables(self, device):
        made = self._tables.get(device)
        if made is None:
            made = self._tables[device] = _Tables(self.layout, self.block, device)
        return made

    def _tables_for_a_launch(self, device):
        made = self.tables(device)
        made.readers.read(device)
        return made

    def __getstate__(self):
        return dict(self.__dict__, _tables=dict())

    def _check(self, q, k, v, softcap, scale, slopes, causal, documents, prefix):
        for name, t in (('q', q), ('k', k), ('v', v)):
            _lib.require_gpu_tensor(t, name)
            if t.dim() != 4:
                raise ValueError('%s must have shape [batch, heads, length, dim]' % name)
            if t.dtype != q.dtype or t.device != q.device:
                raise ValueError('q, k and v must be of one type and on one device')
        if q.dtype not in _lib.DTYPES:
            raise ValueError('Attention supports float16, bfloat16 and float32 (got %s)' % q.dtype)
        Z, H, L, D = q.shape
        kv = k.size(1)
        if D not in (64, 128):
            raise ValueError('head dimensions are 64 and 128 (got %d)' % D)
        if k.shape != v.shape or tuple(k.shape) != (Z, kv, L, D) or kv == 0 or H % kv:
            raise ValueError('q %s, k %s and v %s do not fit together' % (tuple(q.shape), tuple(k.shape), tuple(v.shape)))
        if (L + 64) * D * q.element_size() >= 1 << 32:
            raise ValueError('the rows of a head lie within 4 GiB (got length %d)' % L)
        if H // kv > 127:
            raise ValueError('at most 127 query heads share a key head (got %d)' % (H // kv))
        if k.requires_grad or v.requires_grad:
            self._check_columns(q, k)
        heads, blocks = self.layout.shape[:2]
        if H != heads or -(-L // self.block) != blocks:
            raise ValueError('q %s does not fit a layout of %d heads and %d blocks of %d' % (tuple(q.shape), heads, blocks, self.block))
        check_scores(scale, softcap)
        if prefix is not None and not causal:
            raise ValueError('a prefix needs causal=True')
        for name, t, shape, dtype in (('slopes', slopes, (H,), torch.float32), ('documents', documents, (Z, L), torch.int32), ('prefix', prefix, (Z,), torch.int32)):
            if t is not None and (tuple(t.shape) != shape or t.dtype != dtype or t.device != q.device):
                raise ValueError('%s must be %s %s on %s (got %s %s on %s)' % (name, dtype, list(shape), q.device, t.dtype, list(t.shape), t.device))
        if slopes is not None and slopes.requires_grad and torch.is_grad_enabled():
            raise ValueError('slopes are constants: they get no gradient')

    @staticmethod
    def _check_columns(q, k):
        G, L = q.size(1) // k.size(1), q.size(2)
        if 128 * -(-L // 64) * G >= 1 << 30 and torch.is_grad_enabled():
            raise ValueError('the gradient of a key head reads the rows of fewer than 2^29 positions (got %d query heads of %d)' % (G, L))

    @staticmethod
    def _check_shared(q, k, shared):
        if not isinstance(shared, (tuple, list)) or len(shared) != 2:
            raise ValueError('shared must be a pair of tensors, of the queries and of the keys')
        q_s, k_s = shared
        for t in shared:
            _lib.require_gpu_tensor(t, 'a shared part')
            if t.dtype != q.dtype or t.device != q.device:
                raise ValueError('shared must be of the type of q, k and v, and on their device')
        Z, H, L = q.shape[:3]
        if tuple(q_s.shape) != (Z, H, L, SHARED) or tuple(k_s.shape) != (Z, L, SHARED):
            raise ValueError('shared must be %s and %s (got %s and %s)' % ([Z, H, L, SHARED], [Z, L, SHARED], list(q_s.shape), list(k_s.shape)))
        if Z > 65535:
            raise ValueError('at most 65535 sequences share key parts in a call (got %d)' % Z)

    def __call__(self, q, k, v, scale=1., softcap=0., slopes=None, causal=False, documents=None, prefix=None, shared=None):
        scale, softcap = float(scale), float(softcap or 0.)
        self._check(q, k, v, softcap, scale, slopes, causal, documents, prefix)
        if shared is not None:
            self._check_shared(q, k, shared)
            if shared[1].requires_grad and not (k.requires_grad or v.requires_grad):
                self._check_columns(q, k)
        if q.numel() == 0:
            return torch.empty_like(q) + 0 * (q.sum() + k.sum() + v.sum() + (shared[0].sum() + shared[1].sum() if shared is not None else 0))
        if slopes is not None:
            slopes = slopes.contiguous()
        if prefix is not None:
            prefix = prefix.contiguous()
        if documents is not None and documents.size(1) > 1 and documents.stride(1) != 1:
            documents = documents.contiguous()
        with _lib.on_device(q.device):
            if shared is not None:
                return _shared_rules.apply(q, k, v, *shared, self._tables_for_a_launch(q.device), scale, softcap, slopes, bool(causal), documents, prefix, torch.is_grad_enabled())
            return _rules.apply(q, k, v, self._tables_for_a_launch(q.device), scale, softcap, slopes, bool(causal), documents, prefix, torch.is_grad_enabled())
