"""A cache of latent vectors, and the attention of one new position over it.

In latent attention the keys and values of all heads of a position are made from one vector c (of `latent` elements) and a key part r of 64 that carries the
position and is the same for all heads: k_h = [K_h c ; r], v_h = V_h c.  A prompt or a training step expands them and calls `Attention` with `shared`.  An answer,
position after position, keeps c and r alone, and takes the matrices to the other side: with q_h = [n_h ; t_h] a score is n_h . K_h c + t_h . r = (K_h^T n_h) . c + t_h . r, and the result
is V_h times the sum of the shares' c.  `LatentCache` holds c and r, `LatentAttention` computes what lies between the two products:

    cache = LatentCache(pages, block, latent=512, dtype=torch.bfloat16)
    cache.write(c, r, slots, rotation=rotation, positions=positions)             # c [tokens, latent], r [tokens, 64], turned on the way
    y = LatentAttention(block, layout)(q, q_r, cache, table, lengths, scale=scale)     # q [batch, heads, latent]: K_h^T n_h; q_r [batch, heads, 64]; y [batch, heads, latent]

so that a position takes 2 * (latent + 64) bytes, whatever the number of heads."""
import torch

from . import _lib
from .cache import Pages, check_rotation
from .rules import SHARED, check_scores


class LatentCache(Pages):
    """pages of `block` (16, 32, 64 or 128) positions: a latent vector of 128, 256 or 512 elements and a shared key part of 64, in float16 or bfloat16.  `data` holds
    them, [pages, block, latent + 64] (zeros at first), the shared part behind the latent vector; what a page means to a program, a table of its own says."""

    def __init__(self, pages, block, latent=512, shared=SHARED, dtype=torch.bfloat16, device='cuda'):
        if block not in (16, 32, 64, 128):
            raise ValueError('block must be 16, 32, 64 or 128 (got %s)' % (block,))
        if latent not in (128, 256, 512):
            raise ValueError('latent vectors have 128, 256 or 512 elements (got %s)' % (latent,))
        if shared != SHARED:
            raise ValueError('the shared key part has %d elements (got %s)' % (SHARED, shared))
        if dtype not in (torch.float16, torch.bfloat16):
            raise ValueError('LatentCache holds float16 or bfloat16 (got %s)' % dtype)
        if pages <= 0 or pages * block >= 1 << 31:
            raise ValueError('a cache has at least one page and fewer than 2^31 positions (got %s pages)' % (pages,))
        device = torch.device(device)
        if device.type != 'cuda':
            raise _lib.BlocksparseLibraryError('torch_blocksparse: a cache must live on the GPU (got device %s)' % device)
        if device.index is None:
            device = torch.device('cuda', torch.cuda.current_device())
        self.pages, self.block, self.latent, self.dtype, self.device = int(pages), block, latent, dtype, device
        self.data = torch.zeros((self.pages, block, latent + SHARED), dtype=dtype, device=device)
        self._owner = torch.zeros(self.pages * block, dtype=torch.int32, device=device)     # (zero between calls: bsp_latent_write)
        self._note_users()

    def _operand(self, t, name, tokens, elements):
        if t.device != self.device:
            raise _lib.BlocksparseLibraryError('torch_blocksparse: %s must live on %s (got device %s)' % (name, self.device, t.device))
        if t.dtype != self.dtype or t.shape != (tokens, elements):
            raise ValueError('%s must be %s %s (got %s %s)' % (name, self.dtype, [tokens, elements], t.dtype, list(t.shape)))
        row, one = t.stride()
        if one != 1 or (tokens > 1 and row % 8) or t.data_ptr() % 16:
            t = t.detach().clone(memory_format=torch.contiguous_format)
            row = elements
        return t, (row if tokens > 1 else 0)

    def write(self, c, r, slots, rotation=None, positions=None):
        """Puts c [tokens, latent] and r [tokens, 64] (of the cache's type) at positions slots[t] = page * block + offset, int32.  Tokens with a negative slot, or one past the
        cache, are left out; of tokens with the same slot the last is written.  With a `Rotation` and the tokens' positions [tokens] int32, r is turned on the
        way.  No gradient.  Two writes that run at the same time (on two streams) and have a slot in common leave it as one of them, or part of each."""
        slots = self._check_slots(slots)
        T = slots.numel()
        positions = check_rotation(rotation, positions, T, SHARED, self.device)
        c, c_st = self._operand(c, 'c', T, self.latent)
        r, r_st = self._operand(r, 'r', T, SHARED)
        if T == 0:
            return
        with _lib.on_device(self.device):
            stream = _lib.raw_stream(self.device)
            if stream not in self._users.streams:
                self._users.read(self.device)
            turn = (None, 0, 0, None) if rotation is None else (rotation.fractions(self.device).data_ptr(), rotation.pairs, rotation.neighbours, positions.data_ptr())
            rc = _lib.load().bsp_latent_write(_lib.DTYPES[self.dtype], self.data.data_ptr(), self.pages, self.block, self.latent, c.data_ptr(), c_st, r.data_ptr(), r_st,
                                              slots.data_ptr(), T, self._owner.data_ptr(), *turn, stream)
        _lib.check(rc, 'bsp_latent_write')

    def read(self, slots):
        """(c, r) [tokens, latent] and [tokens, 64] as the cache holds them at slots [tokens]; zeros for slots outside it."""
        slots = self._check_slots(slots)
        c, r = [torch.empty((slots.numel(), n), dtype=self.dtype, device=self.device) for n in (self.latent, SHARED)]
        if slots.numel():
            with _lib.on_device(self.device):
                stream = _lib.raw_stream(self.device)
                if stream not in self._users.streams:
                    self._users.read(self.device)
                rc = _lib.load().bsp_latent_read(_lib.DTYPES[self.dtype], self.data.data_ptr(), self.pages, self.block, self.latent, c.data_ptr(), r.data_ptr(), slots.data_ptr(),
                                                 slots.numel(), stream)
            _lib.check(rc, 'bsp_latent_read')
        return c, r


MOST_ROWS = 2 ** 31 - 1       # places in the table of a layout's rows are 32-bit numbers


def _signed(x):
    return torch.where(x >= 1 << 31, x - (1 << 32), x).to(torch.int32)


def _rows_table(layout, per):
    """what bsp_latent_attention takes of a layout [H, R, C] (host) for units of `per` heads: per unit the block-rows' first entries and the end of the last, then the
    entries (block-column, 64 bits of heads in two ints), which the first entries count from 0"""
    H, R, C = layout.shape
    starts, entries, at = [], [], 0
    for first in range(0, H, per):
        seen = torch.zeros((2, R, C), dtype=torch.int64, device='cpu')
        for i in range(min(per, H - first)):
            seen[i // 32] |= (layout[first + i] != 0).long() << i % 32
        where = torch.nonzero(seen[0] | seen[1])
        counts = torch.bincount(where[:, 0], minlength=R)
        starts.append(torch.cat([torch.zeros(1, dtype=torch.int64, device='cpu'), counts.cumsum(0)]) + at)
        entries.append(torch.stack([where[:, 1], seen[0][where[:, 0], where[:, 1]], seen[1][where[:, 0], where[:, 1]]], 1))
        at += len(where)
    if at > MOST_ROWS:
        raise ValueError('the rows of the layout take %d entries, more than %d' % (at, MOST_ROWS))
    return _signed(torch.cat([torch.cat(starts), torch.cat(entries).flatten(), torch.zeros(3, dtype=torch.int64, device='cpu')]))     # (an entry more: one is read where there is none)


class LatentAttention:
    """Attention of one new position a sequence over a LatentCache, dense or over a block-sparse layout [heads, blocks, blocks].

    Called with q [batch, heads, latent] and q_r [batch, heads, 64] of the cache's type, the cache, the sequences' pages `table` [batch, width] int32 and
    their `lengths` [batch] int32, the new position among them (it is in the cache already).  Position j of sequence b is in page
    table[b, j // block] at offset j % block.  Returns o [batch, heads, latent]:

        y_j = softcap * tanh(scale * (q . c_j + q_r . r_j) / softcap) - slopes[h] * (n - 1 - j),   o = sum_j softmax_j(y_j) c_j      (softcap 0: no cap; else 2^-10 to 1024)

    over j < n = lengths[b], with a layout those in blocks that row (n - 1) // block of head h has.  A page number outside the cache (-1, say) stands for a page that is not
    held: its positions are not seen.  A sequence of length 0, or one that sees nothing, gets zeros.  Lengths count as at most width * block and as at most the
    layout's positions.  A NaN or an infinity in a latent vector that one head sees can reach the others of its sequence.  Sums and shares are fp32; a share is an operand of a product in two
    terms of the cache's type.  No gradient.

    With a layout a table is made at the first call on a device, so a call that is captured into a graph needs one like it before."""

    def __init__(self, block, layout=None):
        if block not in (16, 32, 64, 128):
            raise ValueError('block must be 16, 32, 64 or 128 (got %s)' % (block,))
        if layout is not None and (layout.dim() != 3 or layout.size(1) != layout.size(2) or layout.size(1) > 65535 or layout.numel() == 0):
            raise ValueError('layout must have shape [heads, blocks, blocks], at most 65535 blocks')
        self.block, self.layout = block, layout
        self._rows = dict()

    def __getstate__(self):
        return dict(self.__dict__, _rows=dict())

    def _table(self, device):
        made = self._rows.get(device)
        if made is None:
            layout = self.layout.cpu()
            per = _lib.load().bsp_latent_attention_heads(layout.size(0))
            longest = torch.stack([(layout[h:h + per] != 0).any(0).sum(1) for h in range(0, layout.size(0), per)]).amax(0).cummax(0).values.tolist()   # the most entries of the rows up to each
            made = self._rows[device] = (_rows_table(layout, per).to(device), longest, _lib.Readers())
            made[2].table(made[0])
        return made

    def _fits(self, q, q_r, cache, table, lengths, slopes):
        """whether _refuse has nothing to say of the operands, in as few steps as it takes"""
        if not isinstance(cache, LatentCache):
            return False
        device, dtype, shape, pages = cache.device, cache.dtype, q.shape, table.shape
        if len(shape) != 3 or len(pages) != 2:
            return False
        B, H, D = shape
        return (q.device == device and q_r.device == device and table.device == device and lengths.device == device and q.dtype is dtype and q_r.dtype is dtype and
                table.dtype is torch.int32 and lengths.dtype is torch.int32 and cache.block == self.block and D == cache.latent and q_r.shape == (B, H, SHARED) and 0 < H and B * H < 1 << 24 and
                (self.layout is None or self.layout.shape[0] == H) and pages[0] == B and 0 < pages[1] * self.block < 1 << 24 and lengths.shape == (B,) and
                (slopes is None or (slopes.shape == (H,) and slopes.dtype is torch.float32 and slopes.device == device)))

    def _refuse(self, q, q_r, cache, table, lengths, slopes):
        if not isinstance(cache, LatentCache):
            raise ValueError('LatentAttention reads a LatentCache (got %s)' % type(cache).__name__)
        for name, t in (('q', q), ('q_r', q_r)):
            if t.device != cache.device:
                raise _lib.BlocksparseLibraryError('torch_blocksparse: %s must live on %s, where the cache is (got device %s)' % (name, cache.device, t.device))
            if t.dtype != cache.dtype:
                raise ValueError('%s must be %s, as the cache is (got %s)' % (name, cache.dtype, t.dtype))
        if cache.block != self.block:
            raise ValueError('the cache has pages of %d, the attention blocks of %d' % (cache.block, self.block))
        if q.dim() != 3 or q.size(2) != cache.latent or q.size(1) == 0 or tuple(q_r.shape) != (q.size(0), q.size(1), SHARED):
            raise ValueError('q %s and q_r %s do not fit a cache of latent vectors of %d and a shared part of %d' % (list(q.shape), list(q_r.shape), cache.latent, SHARED))
        B, H = q.shape[:2]
        if B * H >= 1 << 24:
            raise ValueError('a call takes fewer than 2^24 heads of all sequences (got %d)' % (B * H))
        if self.layout is not None and self.layout.size(0) != H:
            raise ValueError('q has %d heads, the layout %d' % (H, self.layout.size(0)))
        if table.dim() != 2 or table.size(0) != B or table.size(1) == 0 or table.dtype != torch.int32 or table.device != q.device:
            raise ValueError('the table of pages must be int32 [%d, width] on %s (got %s %s on %s)' % (B, q.device, table.dtype, list(table.shape), table.device))
        if table.size(1) * self.block >= 1 << 24:
            raise ValueError('a sequence has fewer than 2^24 positions (got a table for %d)' % (table.size(1) * self.block))
        for name, t, shape, dtype in (('lengths', lengths, (B,), torch.int32), ('slopes', slopes, (H,), torch.float32)):
            if (t is not None or name == 'lengths') and (tuple(t.shape) != shape or t.dtype != dtype or t.device != q.device):
                raise ValueError('%s must be %s %s on %s (got %s %s on %s)' % (name, dtype, list(shape), q.device, t.dtype, list(t.shape), t.device))

    def _check(self, q, q_r, cache, table, lengths, scale, softcap, slopes):
        if not self._fits(q, q_r, cache, table, lengths, slopes):
            self._refuse(q, q_r, cache, table, lengths, slopes)
        check_scores(scale, softcap)

    @staticmethod
    def _operand(t):
        (B, H, _), (b, h, one) = t.shape, t.stride()
        if one != 1 or (B > 1 and b % 8) or (H > 1 and h % 8) or t.data_ptr() % 16:
            t = t.detach().clone(memory_format=torch.contiguous_format)
            b, h, one = t.stride()
        return t, (b if B > 1 else 0), (h if H > 1 else 0)

    def __call__(self, q, q_r, cache, table, lengths, scale=1., softcap=0., slopes=None):
        scale, softcap = float(scale), float(softcap or 0.)
        self._check(q, q_r, cache, table, lengths, scale, softcap, slopes)
        B, H, D = q.shape
        device = cache.device
        o = torch.empty_like(q, memory_format=torch.contiguous_format)
        if B == 0:
            return o
        (q, q_sb, q_sh), (q_r, r_sb, r_sh) = self._operand(q), self._operand(q_r)
        width, (next_row, one) = table.shape[1], table.stride()
        if width > 1 and one != 1:
            table = table.contiguous()
            next_row = width
        lengths = lengths.contiguous()
        slopes = slopes.detach().contiguous() if slopes is not None else None
        lib = _lib.load()
        with _lib.on_device(device):
            stream = _lib.raw_stream(device)
            if stream not in cache._users.streams:
                cache._users.read(device)
            rows, blocks, n_rows = None, width, 0
            if self.layout is not None:
                rows, longest, readers = self._table(device)
                if stream not in readers.streams:
                    readers.read(device)
                n_rows = self.layout.shape[1]
                blocks = max(1, longest[min(blocks, n_rows) - 1])
            need = lib.bsp_latent_attention_workspace_bytes(B, H, D, self.block, blocks)
            workspace = torch.empty(need, dtype=torch.uint8, device=device)
            rc = lib.bsp_latent_attention(_lib.DTYPES[q.dtype], q.data_ptr(), q_sb, q_sh, q_r.data_ptr(), r_sb, r_sh, o.data_ptr(), H * D, D, B, H, cache.data.data_ptr(), cache.pages,
                                          self.block, D, table.data_ptr(), next_row if B > 1 else 0, width, lengths.data_ptr(), rows.data_ptr() if rows is not None else None,
                                          n_rows, blocks, scale, softcap, slopes.data_ptr() if slopes is not None else None, workspace.data_ptr(), need, stream)
        _lib.check(rc, 'bsp_latent_attention')
        return o
