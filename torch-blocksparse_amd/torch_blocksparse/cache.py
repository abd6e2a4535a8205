"""A quantised cache of keys and values, and the attention of one new position over it.

A program that answers with a block-sparse model keeps the keys and values of what it has read in pages of `block` positions, which are the
blocks of its layout: `KeyValueCache` holds them in 4 or 8 bits, `CacheAttention` computes a new position's attention over the pages that
its row of the layout names, and reads no other.

    cache = KeyValueCache(pages, block, heads, head_dim, bits=4, device='cuda')
    cache.write(k, v, slots)                           # k, v [tokens, heads, head_dim] to positions page * block + offset
    o = CacheAttention(block, layout)(q, cache, table, lengths, scale=head_dim ** -0.5)     # q, o [batch, query heads, head_dim]

In the cache 32 neighbouring elements of a head share a least value and a step, both float16: least = min x, step = (max x - least) /
(2^bits - 1), and an element is least + code * step with the nearest code (ties to the even one), in exact arithmetic (the step is below zero where the least value is rounded up past all of them).  Elements are taken into
float16's range first; where the rounding of a step takes one past it again, float16 reads 65504 and attention takes a value as 65504.  A group with a NaN reads back as NaN.  A position of a head takes 5 / 8 (4 bits) or 9 / 8 (8 bits) bytes an element.
"""
import torch

from . import _lib
from .rotation import Rotation
from .rules import check_scores


def check_rotation(rotation, positions, tokens, dim, device):
    """the positions [tokens] that a cache is given with a rotation of `dim` elements, as its kernels read them"""
    if rotation is None:
        if positions is not None:
            raise ValueError('positions go with a rotation')
        return None
    if not isinstance(rotation, Rotation):
        raise ValueError('rotation must be a Rotation (got %s)' % type(rotation).__name__)
    if 2 * rotation.pairs > dim:
        raise ValueError('a rotation of %d pairs does not fit %d elements' % (rotation.pairs, dim))
    if positions is None:
        raise ValueError('a rotation needs positions')
    rotation.check_positions(positions, ((tokens,),), device)
    return positions.contiguous()


class Pages:
    """what the caches of this package have in common: positions in pages, named by slots, written by whatever stream is current"""

    def _note_users(self):
        self._users = _lib.Readers()                       # (the streams of all calls: memory that is given back while one writes it would change under its next owner)
        self._users.table(self.data, self._owner)

    def __getstate__(self):
        return {n: x for n, x in self.__dict__.items() if n != '_users'}

    def __setstate__(self, state):
        self.__dict__.update(state)
        self._note_users()

    def _check_slots(self, slots):
        if slots.dim() != 1 or slots.dtype != torch.int32 or slots.device != self.device:
            raise ValueError('slots must be a vector of int32 on %s (got %s %s on %s)' % (self.device, slots.dtype, list(slots.shape), slots.device))
        if slots.numel() >= 1 << 24:
            raise ValueError('a call takes fewer than 2^24 tokens (got %d)' % slots.numel())
        return slots.contiguous()


class KeyValueCache(Pages):
    """pages of `block` (16, 32, 64 or 128) positions of `heads` key heads of 64 or 128 elements, in 4 or 8 bits.  `data` holds the pages
    ([pages, bytes of a page]; zeros at first, which stand for zeros); what a page means to a program, a table of its own says."""

    def __init__(self, pages, block, heads, head_dim, bits=4, device='cuda'):
        if block not in (16, 32, 64, 128):
            raise ValueError('block must be 16, 32, 64 or 128 (got %s)' % (block,))
        if bits not in (4, 8):
            raise ValueError('bits must be 4 or 8 (got %s)' % (bits,))
        if head_dim not in (64, 128):
            raise ValueError('head dimensions are 64 and 128 (got %s)' % (head_dim,))
        if heads <= 0 or pages <= 0 or pages * block >= 1 << 31:
            raise ValueError('a cache has at least one page and head and fewer than 2^31 positions (got %s pages, %s heads)' % (pages, heads))
        device = torch.device(device)
        if device.type != 'cuda':
            raise _lib.BlocksparseLibraryError('torch_blocksparse: a cache must live on the GPU (got device %s)' % device)
        if device.index is None:
            device = torch.device('cuda', torch.cuda.current_device())
        self.pages, self.block, self.heads, self.head_dim, self.bits, self.device = int(pages), block, int(heads), head_dim, bits, device
        self.data = torch.zeros((self.pages, _lib.load().bsp_cache_page_bytes(block, self.heads, head_dim, bits)), dtype=torch.uint8, device=device)
        self._owner = torch.zeros(self.pages * block, dtype=torch.int32, device=device)     # (zero between calls: bsp_cache_write)
        self._note_users()

    def _operand(self, t, name, tokens):
        if t.device != self.device:
            raise _lib.BlocksparseLibraryError('torch_blocksparse: %s must live on %s (got device %s)' % (name, self.device, t.device))
        if t.dtype not in _lib.DTYPES:
            raise ValueError('KeyValueCache takes float16, bfloat16 and float32 (got %s)' % t.dtype)
        if t.shape != (tokens, self.heads, self.head_dim):
            raise ValueError('%s must be %s (got %s)' % (name, [tokens, self.heads, self.head_dim], list(t.shape)))
        unit, (row, head, one) = 16 // t.element_size(), t.stride()
        if one != 1 or (tokens > 1 and row % unit) or (self.heads > 1 and head % unit) or t.data_ptr() % 16:
            t = t.detach().clone(memory_format=torch.contiguous_format)
            row, head, one = t.stride()
        return t, (row if tokens > 1 else 0), (head if self.heads > 1 else 0)

    def write(self, k, v, slots, rotation=None, positions=None):
        """Quantises k and v [tokens, heads, head_dim] (of one type) into positions slots[t] = page * block + offset of the cache.  Tokens with a
        negative slot, or one past the cache, are left out; of tokens with the same slot the last is written.  No gradient.  Two writes that run at
        the same time (on two streams) and have a slot in common leave it as one of them, or half of each.

        With a `Rotation` and the tokens' positions [tokens] int32 the keys are turned on the way, in 64 bits and with no rounding before their codes (so a NaN or an infinity makes
        its pair's other element one too); what `rotation(k, positions=positions)` gives is rounded to the type of k."""
        slots = self._check_slots(slots)
        T = slots.numel()
        positions = check_rotation(rotation, positions, T, self.head_dim, self.device)
        k, k_st, k_sh = self._operand(k, 'k', T)
        v, v_st, v_sh = self._operand(v, 'v', T)
        if k.dtype != v.dtype:
            raise ValueError('k and v must be of one type (got %s and %s)' % (k.dtype, v.dtype))
        if T == 0:
            return
        with _lib.on_device(self.device):
            stream = _lib.raw_stream(self.device)
            if stream not in self._users.streams:
                self._users.read(self.device)
            args = (_lib.DTYPES[k.dtype], self.data.data_ptr(), self.pages, self.block, self.heads, self.head_dim, self.bits, k.data_ptr(), k_st, k_sh,
                    v.data_ptr(), v_st, v_sh, slots.data_ptr(), T, self._owner.data_ptr())
            if rotation is None:
                rc = _lib.load().bsp_cache_write(*args, stream)
            else:
                rc = _lib.load().bsp_cache_write_rotated(*args, rotation.fractions(self.device).data_ptr(), rotation.pairs, rotation.neighbours, positions.data_ptr(), stream)
        _lib.check(rc, 'bsp_cache_write')

    def read(self, slots, dtype=torch.float16):
        """(k, v) [tokens, heads, head_dim] as the cache holds them at slots [tokens]; zeros for slots outside it."""
        slots = self._check_slots(slots)
        if dtype not in _lib.DTYPES:
            raise ValueError('KeyValueCache gives float16, bfloat16 and float32 (got %s)' % dtype)
        k = torch.empty((slots.numel(), self.heads, self.head_dim), dtype=dtype, device=self.device)
        v = torch.empty_like(k)
        if slots.numel():
            with _lib.on_device(self.device):
                stream = _lib.raw_stream(self.device)
                if stream not in self._users.streams:
                    self._users.read(self.device)
                rc = _lib.load().bsp_cache_read(_lib.DTYPES[dtype], self.data.data_ptr(), self.pages, self.block, self.heads, self.head_dim, self.bits, k.data_ptr(),
                                                v.data_ptr(), slots.data_ptr(), slots.numel(), stream)
            _lib.check(rc, 'bsp_cache_read')
        return k, v


MOST_ROWS = 2 ** 31 - 1       # places in the table of a layout's rows are 32-bit numbers


def _rows_table(layout, kv_heads):
    """what bsp_cache_attention takes of a layout [H, R, C] (host): per unit of query heads the block-rows' first entries, then the entries"""
    H, R, C = layout.shape
    G = H // kv_heads
    per = -(-G // -(-G // 16))
    units = [(g * G + u, min(per, G - u)) for g in range(kv_heads) for u in range(0, G, per)]
    starts, entries, at = [], [], len(units) * (R + 1)
    for first, n in units:
        seen = torch.zeros((R, C), dtype=torch.int64, device='cpu')
        for i in range(n):
            seen |= (layout[first + i] != 0).long() << i
        where = torch.nonzero(seen)
        counts = torch.bincount(where[:, 0], minlength=R)
        starts.append(torch.cat([torch.zeros(1, dtype=torch.int64, device='cpu'), counts.cumsum(0)]) + at)
        entries.append((where[:, 1] << 16) | seen[where[:, 0], where[:, 1]])
        at += len(where)
    if at > MOST_ROWS:
        raise ValueError('the rows of the layout take %d entries, more than %d' % (at, MOST_ROWS))
    table = torch.cat(starts + entries)
    return torch.where(table >= 1 << 31, table - (1 << 32), table).to(torch.int32), int((layout != 0).any(0).sum(1).max()) if R else 0


class CacheAttention:
    """Attention of one new position a sequence over a KeyValueCache, dense or over a block-sparse layout [query heads, blocks, blocks].

    Called with q [batch, query heads, head_dim] (float16 or bfloat16), the cache, the sequences' pages `table` [batch, width] int32 and
    their `lengths` [batch] int32, the new position among them (its key and value are in the cache already).  Position j of sequence b is in page
    table[b, j // block] at offset j % block.  Returns o [batch, query heads, head_dim]:

        y_j = softcap * tanh(scale * q . k_j / softcap) - slopes[h] * (n - 1 - j),   o = sum_j softmax_j(y_j) v_j      (softcap 0: no cap; else 2^-10 to 1024)

    over j < n = lengths[b], with a layout those in blocks that row (n - 1) // block of head h has: what `Attention` with causal=True gives for its last
    row.  A page number outside the cache (-1, say) stands for a page that is not held: its positions are not seen, so pages that no later
    row of the layout names can be given to others.  A sequence of length 0, or one that sees nothing, gets zeros.  Lengths count as
    at most width * block and as at most the layout's positions.  A NaN in a value that one query head of a key head sees can reach its other query heads.  Query head h uses key head h // (query heads / key heads).  No gradient.

    With a layout a table is made at the first call for a number of key heads on a device, so a call that is captured into a graph needs one like it
    before."""

    def __init__(self, block, layout=None):
        if block not in (16, 32, 64, 128):
            raise ValueError('block must be 16, 32, 64 or 128 (got %s)' % (block,))
        if layout is not None and (layout.dim() != 3 or layout.size(1) != layout.size(2) or layout.size(1) > 65535 or layout.numel() == 0):
            raise ValueError('layout must have shape [heads, blocks, blocks], at most 65535 blocks')
        self.block, self.layout = block, layout
        self._rows = dict()

    def __getstate__(self):
        return dict(self.__dict__, _rows=dict())

    def _table(self, kv_heads, device):
        made = self._rows.get((kv_heads, device))
        if made is None:
            layout = self.layout.cpu()
            longest = (layout != 0).any(0).sum(1).cummax(0).values.tolist()       # the most entries of the rows up to each
            made = self._rows[kv_heads, device] = (_rows_table(layout, kv_heads)[0].to(device), longest, _lib.Readers())
            made[2].table(made[0])
        return made

    def _check(self, q, cache, table, lengths, scale, softcap, slopes):
        if q.device != cache.device:
            raise _lib.BlocksparseLibraryError('torch_blocksparse: q must live on %s, where the cache is (got device %s)' % (cache.device, q.device))
        if q.dtype not in (torch.float16, torch.bfloat16):
            raise ValueError('CacheAttention supports float16 and bfloat16 (got %s)' % q.dtype)
        if not isinstance(cache, KeyValueCache):
            raise ValueError('CacheAttention reads a KeyValueCache (got %s)' % type(cache).__name__)
        if cache.block != self.block:
            raise ValueError('the cache has pages of %d, the attention blocks of %d' % (cache.block, self.block))
        if q.dim() != 3 or q.size(2) != cache.head_dim or q.size(1) == 0 or q.size(1) % cache.heads:
            raise ValueError('q %s does not fit a cache of %d heads of %d' % (list(q.shape), cache.heads, cache.head_dim))
        B, H = q.shape[:2]
        if self.layout is not None and self.layout.size(0) != H:
            raise ValueError('q has %d heads, the layout %d' % (H, self.layout.size(0)))
        if table.dim() != 2 or table.size(0) != B or table.size(1) == 0 or table.dtype != torch.int32 or table.device != q.device:
            raise ValueError('the table of pages must be int32 [%d, width] on %s (got %s %s on %s)' % (B, q.device, table.dtype, list(table.shape), table.device))
        if table.size(1) * self.block >= 1 << 24:
            raise ValueError('a sequence has fewer than 2^24 positions (got a table for %d)' % (table.size(1) * self.block))
        for name, t, shape, dtype in (('lengths', lengths, (B,), torch.int32), ('slopes', slopes, (H,), torch.float32)):
            if (t is not None or name == 'lengths') and (tuple(t.shape) != shape or t.dtype != dtype or t.device != q.device):
                raise ValueError('%s must be %s %s on %s (got %s %s on %s)' % (name, dtype, list(shape), q.device, t.dtype, list(t.shape), t.device))
        check_scores(scale, softcap)

    def __call__(self, q, cache, table, lengths, scale=1., softcap=0., slopes=None):
        scale, softcap = float(scale), float(softcap or 0.)
        self._check(q, cache, table, lengths, scale, softcap, slopes)
        B, H, D = q.shape
        q = q.detach()
        o = torch.empty((B, H, D), dtype=q.dtype, device=q.device)
        if B == 0:
            return o
        if q.stride(2) != 1 or (B > 1 and q.stride(0) % 8) or (H > 1 and q.stride(1) % 8) or q.data_ptr() % 16:
            q = q.clone(memory_format=torch.contiguous_format)
        if table.size(1) > 1 and table.stride(1) != 1:
            table = table.contiguous()
        lengths = lengths.contiguous()
        slopes = slopes.detach().contiguous() if slopes is not None else None
        lib = _lib.load()
        with _lib.on_device(q.device):
            stream = _lib.raw_stream(q.device)
            if stream not in cache._users.streams:
                cache._users.read(q.device)
            rows, blocks, n_rows = None, table.size(1), 0
            if self.layout is not None:
                rows, longest, readers = self._table(cache.heads, q.device)
                if stream not in readers.streams:
                    readers.read(q.device)
                n_rows = self.layout.size(1)
                blocks = max(1, min(blocks, longest[min(blocks, n_rows) - 1]))
            splits = lib.bsp_cache_attention_splits(B, H, cache.heads, self.block, blocks)
            need = lib.bsp_cache_attention_workspace_bytes(B, H, cache.heads, D, splits)
            workspace = torch.empty(need, dtype=torch.uint8, device=q.device) if need else None
            rc = lib.bsp_cache_attention(_lib.DTYPES[q.dtype], q.data_ptr(), q.stride(0) if B > 1 else 0, q.stride(1) if H > 1 else 0, o.data_ptr(), H * D, D, B, H,
                                         cache.data.data_ptr(), cache.pages, self.block, cache.heads, D, cache.bits, table.data_ptr(), table.stride(0) if B > 1 else 0,
                                         table.size(1), lengths.data_ptr(), rows.data_ptr() if rows is not None else None, n_rows, blocks, scale, softcap,
                                         slopes.data_ptr() if slopes is not None else None, workspace.data_ptr() if need else None, need, splits,
                                         stream)
            _lib.check(rc, 'bsp_cache_attention')
        return o
