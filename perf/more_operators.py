"""Rotated positions, rotated appends to paged caches and latent attention in both forms: the work that they are measured on.

Operators that follow each other in a program that trains a model with rotated positions, or with keys and values made from one latent
vector a token, and then answers with it:
  rotate      torch_blocksparse.Rotation: pairs of elements turned by position times frequency, of queries and keys in one call; forward, and
              forward with the gradients
  append      KeyValueCache.write with a rotation: keys turned on the way to their codes in the pages; and LatentCache.write, which puts latent
              vectors and the turned key part that all heads share into its pages
  latent      torch_blocksparse.LatentAttention: the attention of one new token a sequence over a LatentCache, keys and values being the
              latent vectors themselves (the absorbed form)
  expanded    torch_blocksparse.Attention with a key part that all heads share beside the heads' own (the expanded form); forward, and forward
              with the gradients of all five operands

listed() gives the named cases, draw(rng) one more of the same ranges, prepare() what a program holds before the call, run() one
pass (own False: elementary torch operations; own True: the package's operators), work() what a pass cannot do without, exact()
the results in 64 bits."""
import math
import os
import sys

import numpy as np
import torch

own = False

_DTYPES = {'fp16': torch.float16, 'bf16': torch.bfloat16, 'fp32': torch.float32}
_SIZE = {'fp16': 2, 'bf16': 2, 'fp32': 4}
_GROUP = 32                                        # values that share a scale and a least value in a quantised cache
_SHARED = 64                                       # elements of the key part that all heads share


def _package():
    path = os.path.abspath('torch-blocksparse_amd')
    if path not in sys.path:
        sys.path.insert(0, path)
    import torch_blocksparse
    return torch_blocksparse


# ---- cases ----------------------------------------------------------------------------------------------------------------------


def _rotate(dtype, Z, H, kv, L, d, turned, neighbours, train, base=10000.):
    """L 0: a decoding step, one token for each of Z sequences"""
    return dict(op='rotate', dtype=dtype, batch=Z, heads=H, kv_heads=kv, length=L, dim=d, turned=turned, neighbours=neighbours, train=train, base=base)


def _append(dtype, tokens, heads, d, turned, block, bits, neighbours=False, base=10000.):
    return dict(op='append', dtype=dtype, tokens=tokens, heads=heads, dim=d, turned=turned, block=block, bits=bits, neighbours=neighbours, base=base)


def _append_latent(dtype, tokens, latent, block, neighbours=True, base=10000.):
    return dict(op='append', dtype=dtype, tokens=tokens, heads=0, dim=latent, turned=_SHARED, block=block, bits=16, neighbours=neighbours, base=base)


def _latent(dtype, batch, H, L, latent, block, layout='none', **options):
    c = dict(op='latent', dtype=dtype, batch=batch, heads=H, length=L, latent=latent, block=block, layout=layout, softcap=0., slopes=False)
    c.update(options)
    return c


def _expanded(dtype, Z, H, L, d, block, layout, **options):
    c = dict(op='expanded', dtype=dtype, batch=Z, heads=H, length=L, dim=d, block=block, layout=layout, train=True, causal=True, softcap=0., documents=0, prefix=False)
    c.update(options)
    return c


def listed():
    cases = []

    def case(name, c):
        cases.append(dict(c, name=name))

    # The queries and keys of a decoding step, sixteen sequences, each at a position of its own: launches and the call are what counts.
    case('rotate_step', _rotate('bf16', 16, 32, 8, 0, 128, 128, False, False))
    # The queries and keys of a training step at full length, key heads shared by four query heads.
    case('rotate_train', _rotate('bf16', 4, 32, 8, 4096, 128, 128, False, True))
    # Single precision, half of each head turned, pairs of neighbouring elements, a ragged length.
    case('rotate_train_fp32_part', _rotate('fp32', 2, 12, 12, 2023, 64, 32, True, True))
    # A decoding step's new keys and values, one token for each of eight sequences.
    case('append_step_4bit', _append('bf16', 8, 16, 64, 64, 64, 4))
    # The keys and values of a long prompt.
    case('append_prompt_8bit', _append('fp16', 16384, 8, 128, 128, 64, 8, base=500000.))
    # A prompt of odd length into a cache of latent vectors.
    case('append_latent_prompt', _append_latent('bf16', 20011, 512, 64))
    # The first tokens of one answer.
    case('latent_short', _latent('fp16', 1, 16, 33, 512, 16))
    # Sixteen sequences that a block-sparse layout was trained on, capped scores.
    case('latent_layout', _latent('fp16', 16, 16, 4096, 512, 64, 'fixed512', softcap=20.))
    # Long sequences of uneven length under many heads: the cache's bytes, and the products of all heads with them.
    case('latent_long', _latent('bf16', 16, 128, 16384, 512, 64))
    # One short prompt in a training loop's last, ragged batch.
    case('expanded_short', _expanded('fp16', 1, 4, 57, 64, 16, 'dense'))
    # Documents packed into rows of a length that is no multiple of anything.
    case('expanded_train', _expanded('bf16', 2, 16, 4001, 128, 64, 'dense', documents=5))
    # The prompt of a request, answered without gradients.
    case('expanded_prompt', _expanded('bf16', 1, 16, 8192, 128, 64, 'dense', train=False))
    return cases


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(['rotate', 'append', 'append', 'latent', 'latent', 'expanded', 'expanded'])
    dtype = rng.choice(['fp16', 'bf16', 'bf16', 'fp32'])
    d = rng.choice([64, 64, 128])
    base = rng.choice([10000., 10000., 500000.])
    if op == 'rotate':
        kv, group, Z = rng.choice([1, 2, 3, 8]), rng.choice([1, 2, 4]), rng.choice([1, 1, 2, 4])
        step = rng.random() < 0.3
        return _rotate(dtype, _log(rng, 1, 300) if step else Z, kv * group, kv, 0 if step else _log(rng, 1, 16384 // Z), d, rng.choice([d, d, d // 2, 16, 48]),
                       rng.random() < 0.5, not step and rng.random() < 0.7, base)
    if op == 'append':
        tokens, block, neighbours = _log(rng, 1, 16000), rng.choice([16, 32, 64, 128]), rng.random() < 0.5
        if rng.random() < 0.4:
            return _append_latent(rng.choice(['fp16', 'bf16']), tokens, rng.choice([128, 256, 512, 512]), block, neighbours, base)
        return _append(dtype, tokens, rng.choice([1, 2, 3, 8]), d, rng.choice([d, d, d // 2, 48]), block, rng.choice([4, 8]), neighbours, base)
    if op == 'latent':
        dtype, H = rng.choice(['fp16', 'bf16']), rng.choice([1, 5, 8, 16, 16, 24, 32, 64, 96, 128])
        batch = _log(rng, 1, 96)
        L = _log(rng, 1, min(32768, 262144 // batch))
        layout = rng.choice(['none', 'none', 'fixed256', 'bigbird']) if H <= 32 else 'none'
        block = rng.choice([16, 32, 64, 128])
        if layout != 'none':                           # (a layout of every pair of blocks is made on the host)
            L, block = min(L, 8192), max(block, 32)
        return _latent(dtype, batch, H, L, rng.choice([512, 512, 512, 256, 128]), block, layout, softcap=rng.choice([0., 0., 30.]), slopes=rng.random() < 0.25)
    train = rng.random() < 0.7
    # (a lone position's gradients are zero and what rounding leaves of them, so nothing to compare: training begins at 16)
    L = _log(rng, 16 if train else 1, 8192 if dtype != 'fp32' else 3000)
    most = max(1, int((2e7 if dtype == 'fp32' else 1.4e8) // (L * L)))                  # heads of all sequences
    H = min(rng.choice([1, 2, 3, 8, 16]), most)
    Z = min(rng.choice([1, 1, 2, 4]), max(1, most // H))
    causal = rng.random() < 0.8
    return _expanded(dtype, Z, H, L, d, rng.choice([16, 32, 64, 128]), rng.choice(['dense', 'dense', 'fixed128', 'bigbird']), causal=causal, train=train,
                     softcap=rng.choice([0., 0., 0., 30.]), documents=min(rng.choice([0, 0, 1, 3, 9]), L // 8), prefix=causal and rng.random() < 0.25)


# ---- what the cases hold ----------------------------------------------------------------------------------------------------------


def _layout(kind, H, blocks, block, causal):
    """[H, blocks, blocks] of zeros and ones: every block ('dense'), windows of n positions and their last blocks ('fixed<n>'), or a
    band of three block-columns, two global ones and three random ones a row ('bigbird'); causal: no block above the diagonal"""
    i = np.arange(blocks)
    if kind == 'dense':
        lay = np.ones((H, blocks, blocks), bool)
    elif kind.startswith('fixed'):
        n = max(1, int(kind[5:]) // block)
        lay = np.repeat(((i[:, None] // n == i[None, :] // n) | (i[None, :] % n == n - 1))[None], H, 0)
    else:
        lay = np.repeat(((abs(i[:, None] - i[None, :]) <= 2) | (i[None, :] < 2))[None], H, 0)
        r = np.random.RandomState(blocks)
        for _ in range(3):
            pick = (r.rand(H, blocks) * (i + 1 if causal else blocks)).astype(int)
            np.put_along_axis(lay, pick[:, :, None], True, 2)
    if causal:
        lay &= i[None, :] <= i[:, None]
    return lay


def _documents(case):
    """[Z, L] ids: the positions of a row in pieces of uneven length, and some at the end that belong to none (-1)"""
    Z, L, n = case['batch'], case['length'], case['documents']
    r = np.random.RandomState(L + 31 * n)
    ids = np.empty((Z, L), np.int32)
    for z in range(Z):
        end = L - int(r.rand() * L / 8)
        cuts = np.sort(r.randint(0, max(1, end), n - 1))
        ids[z] = np.searchsorted(cuts, np.arange(L), side='right')
        ids[z, end:] = -1
    return ids


def _prefix(case):
    Z, L = case['batch'], case['length']
    return ((np.arange(Z) + 1) * L // (4 * Z)).astype(np.int32)


def _lengths(case):
    """positions of each sequence, from the longest down to a quarter of it"""
    B, L = case['batch'], case['length']
    return np.maximum(1, L - (np.arange(B) * 7 % B) * (3 * L // 4) // max(1, B)).astype(np.int32)


def _frequencies(case):
    """radians a position of each pair, in 64 bits"""
    n = case['turned'] // 2
    return torch.tensor([case['base'] ** (-i / n) for i in range(n)], dtype=torch.float64)


def _slopes(H):
    return torch.tensor([2. ** (-8. * (h + 1) / H) for h in range(H)])


def _generator(seed):
    return torch.Generator(device='cuda').manual_seed(seed)


def _randn(shape, dtype, g, scale=1.):
    return (torch.randn(shape, device='cuda', generator=g) * scale).to(dtype)


def _inputs(case, seed):
    """the tensors of a case"""
    g, dtype, op = _generator(seed), _DTYPES[case['dtype']], case['op']
    if op == 'rotate':
        Z, H, kv, L, d = [case[n] for n in ('batch', 'heads', 'kv_heads', 'length', 'dim')]
        if L == 0:
            return dict(q=_randn((Z, H, d), dtype, g), k=_randn((Z, kv, d), dtype, g), positions=torch.randint(0, 131072, (Z,), device='cuda', generator=g, dtype=torch.int32))
        starts = torch.randint(0, 32768, (Z, 1), device='cuda', generator=g, dtype=torch.int32)              # each sequence goes on from where it was
        x = dict(q=_randn((Z, H, L, d), dtype, g), k=_randn((Z, kv, L, d), dtype, g), positions=starts + torch.arange(L, device='cuda', dtype=torch.int32))
        if case['train']:
            x.update(dq=_randn((Z, H, L, d), dtype, g), dk=_randn((Z, kv, L, d), dtype, g))
        return x
    if op == 'append':
        T, H, d, block = case['tokens'], case['heads'], case['dim'], case['block']
        pages = (T + block - 1) // block + 3               # pages anywhere, filled from their first position on
        slots = (torch.randperm(pages, device='cuda', generator=g)[:, None] * block + torch.arange(block, device='cuda')).flatten()[:T].int()
        positions = torch.randint(0, 131072 - T, (1,), device='cuda', generator=g, dtype=torch.int32) + torch.arange(T, device='cuda', dtype=torch.int32)
        if H:
            return dict(k=_randn((T, H, d), dtype, g, 1.5), v=_randn((T, H, d), dtype, g), slots=slots, positions=positions, pages=pages)
        return dict(c=_randn((T, d), dtype, g), r=_randn((T, _SHARED), dtype, g, 1.5), slots=slots, positions=positions, pages=pages)
    if op == 'latent':
        B, H, block, latent = case['batch'], case['heads'], case['block'], case['latent']
        width = (case['length'] + block - 1) // block
        pages = B * width + 2
        # (scores of a few units: what scaled products of trained models have)
        return dict(c=_randn((pages * block, latent), dtype, g), r=_randn((pages * block, _SHARED), dtype, g), pages=pages,
                    table=torch.randperm(pages, device='cuda', generator=g)[:B * width].int().view(B, width),
                    q=_randn((B, H, latent), dtype, g), qr=_randn((B, H, _SHARED), dtype, g, 1.5))
    Z, H, L, d = [case[n] for n in ('batch', 'heads', 'length', 'dim')]
    scale = 2. if case['softcap'] else 1.
    x = dict(q=_randn((Z, H, L, d), dtype, g, scale), k=_randn((Z, H, L, d), dtype, g), v=_randn((Z, H, L, d), dtype, g),
             qr=_randn((Z, H, L, _SHARED), dtype, g, scale), kr=_randn((Z, L, _SHARED), dtype, g))
    if case['train']:
        x.update(do=_randn((Z, H, L, d), dtype, g))
    return x


def _quantised(x, bits):
    """[.., d] -> codes [.., d] (uint8), scale and least value [.., d / 32] (fp16).  The value nearest a code's border decides, so in 64 bits."""
    x = x.double().unflatten(-1, (-1, _GROUP)).clamp(-65504., 65504.)
    low = x.amin(-1).half()
    scale = ((x.amax(-1) - low.double()) / (2 ** bits - 1)).half()
    s = scale.double()[..., None]
    codes = torch.where(s > 0, ((x - low.double()[..., None]) / torch.where(s > 0, s, 1.)).round().clamp(0, 2 ** bits - 1), 0.)
    return codes.to(torch.uint8).flatten(-2), scale, low


def prepare(case, seed):
    state = dict(_inputs(case, seed), case=case, dtype=_DTYPES[case['dtype']])
    op = case['op']
    if op in ('rotate', 'append'):
        frequencies = _frequencies(case)
        if own:
            state['rotation'] = _package().Rotation(frequencies, neighbours=case['neighbours'])
        else:
            state['frequencies'] = frequencies.cuda()
    if op == 'rotate':
        if own and case['train']:
            state.update(q=state['q'].requires_grad_(True), k=state['k'].requires_grad_(True))
    elif op == 'append':
        rows, H, d = state['pages'] * case['block'], case['heads'], case['dim']
        if own:
            tb = _package()
            state['cache'] = tb.KeyValueCache(state['pages'], case['block'], H, d, bits=case['bits'], device='cuda') if H else \
                tb.LatentCache(state['pages'], case['block'], d, _SHARED, dtype=state['dtype'], device='cuda')
        elif H:                                            # the codes of a key and of a value (two to a byte in 4 bits), scales and least values
            state['held'] = [(torch.zeros((rows, H, d * case['bits'] // 8), dtype=torch.uint8, device='cuda'),
                              torch.zeros((rows, H, d // _GROUP), dtype=torch.float16, device='cuda'), torch.zeros((rows, H, d // _GROUP), dtype=torch.float16, device='cuda'))
                             for _ in range(2)]
        else:
            state['held'] = torch.zeros((state['pages'], case['block'], d + _SHARED), dtype=state['dtype'], device='cuda')
    elif op == 'latent':
        B, H, block = case['batch'], case['heads'], case['block']
        state['lengths'] = torch.from_numpy(_lengths(case)).cuda()
        state['slopes'] = _slopes(H).cuda() if case['slopes'] else None
        layout = None if case['layout'] == 'none' else torch.from_numpy(_layout(case['layout'], H, state['table'].size(1), block, True))
        c, r = state.pop('c'), state.pop('r')
        if own:
            tb = _package()
            state['cache'] = tb.LatentCache(state['pages'], block, case['latent'], _SHARED, dtype=state['dtype'], device='cuda')
            state['cache'].write(c, r, torch.arange(c.size(0), device='cuda', dtype=torch.int32))
            state['op'] = tb.LatentAttention(block, None if layout is None else layout.long())
        else:
            state['held'] = torch.cat([c, r], 1)
            state['layout'] = None if layout is None else layout.cuda()
    else:
        L, block = case['length'], case['block']
        layout = torch.from_numpy(_layout(case['layout'], case['heads'], (L + block - 1) // block, block, case['causal'] and not case['prefix']))
        state.update(documents=torch.from_numpy(_documents(case)).cuda() if case['documents'] else None,
                     prefix=torch.from_numpy(_prefix(case)).cuda() if case['prefix'] else None)
        if own:
            state['op'] = _package().Attention(layout.long(), block)
            if case['train']:
                state.update({n: state[n].requires_grad_(True) for n in ('q', 'k', 'v', 'qr', 'kr')})
        else:
            state['layout'] = layout.cuda()
    return state


# ---- one pass -------------------------------------------------------------------------------------------------------------------


def run(state):
    return {'rotate': _run_rotate, 'append': _run_append, 'latent': _run_latent, 'expanded': _run_expanded}[state['case']['op']](state)


def _turn(x, angles, neighbours, back=False):
    """x with the pairs of its first 2 n elements turned by angles [.., n] (in 64 bits, as far positions need): elements i and n + i, or 2 i and 2 i + 1"""
    cos, sin = angles.cos().to(x.dtype), angles.sin().to(x.dtype)
    if back:
        sin = -sin
    n = angles.size(-1)
    a, b = (x[..., 0:2 * n:2], x[..., 1:2 * n:2]) if neighbours else (x[..., :n], x[..., n:2 * n])
    y, z = a * cos - b * sin, a * sin + b * cos
    turned = torch.stack((y, z), -1).flatten(-2) if neighbours else torch.cat((y, z), -1)
    return torch.cat((turned, x[..., 2 * n:]), -1)


def _run_rotate(state):
    case, q, k, positions = state['case'], state['q'], state['k'], state['positions']
    if own:
        if not case['train']:
            return state['rotation'](q, k, positions=positions)
        y, z = state['rotation'](q, k, positions=positions)
        return (y.detach(), z.detach()) + torch.autograd.grad((y, z), (q, k), (state['dq'], state['dk']))
    angles = (positions.double()[..., None] * state['frequencies']).unsqueeze(-2 if case['length'] == 0 else 1)
    out = [(q, False), (k, False)] + ([(state['dq'], True), (state['dk'], True)] if case['train'] else [])
    return tuple(_turn(x.float(), angles, case['neighbours'], back).to(x.dtype) for x, back in out)


def _run_append(state):
    case, slots = state['case'], state['slots']
    if own:
        if not case['heads']:
            state['cache'].write(state['c'], state['r'], slots, rotation=state['rotation'], positions=state['positions'])
            return state['cache'].data
        state['cache'].write(state['k'], state['v'], slots, rotation=state['rotation'], positions=state['positions'])
        return state['cache'].read(slots, state['dtype'])
    angles = state['positions'].double()[:, None] * state['frequencies']
    at = slots.long()
    if not case['heads']:
        r = _turn(state['r'].float(), angles, case['neighbours']).to(state['dtype'])
        state['held'].view(-1, case['dim'] + _SHARED)[at] = torch.cat((state['c'], r), 1)
        return state['held']
    k, bits = _turn(state['k'].double(), angles[:, None], case['neighbours']), case['bits']             # (in 64 bits: values next to a code's border)
    return tuple(_written(held, x, at, bits).to(state['dtype']) for held, x in zip(state['held'], (k, state['v'])))


def _written(held, x, at, bits):
    """x into what is held of a cache, and the values, in 32 bits, that it then has there"""
    codes, scale, low = _quantised(x, bits)
    held[0][at] = codes[..., 0::2] | codes[..., 1::2] << 4 if bits == 4 else codes
    held[1][at], held[2][at] = scale, low
    codes, scale, low = [t[at] for t in held]
    if bits == 4:
        codes = torch.stack((codes & 15, codes >> 4), -1).flatten(-2)
    return (codes.float().unflatten(-1, (-1, _GROUP)) * scale.float()[..., None] + low.float()[..., None]).flatten(-2)


def _run_latent(state):
    case, q, qr, table, lengths = state['case'], state['q'], state['qr'], state['table'], state['lengths']
    latent, block, cap = case['latent'], case['block'], case['softcap']
    scale = (128 + _SHARED) ** -0.5                     # of the expanded heads that the queries were absorbed from
    if own:
        return state['op'](q, qr, state['cache'], table, lengths, scale=scale, softcap=cap, slopes=state['slopes'])
    at = (table.long()[:, :, None] * block + torch.arange(block, device='cuda')).flatten(1)              # [B, positions]
    x = state['held'][at].float()                       # [B, positions, latent + 64]
    logits = torch.matmul(torch.cat((q, qr), -1).float(), x.transpose(-1, -2)).mul_(scale)
    if cap:
        logits = logits.div_(cap).tanh_().mul_(cap)
    j = torch.arange(at.size(1), device='cuda')
    last = lengths.long() - 1
    if case['slopes']:
        logits = logits - state['slopes'][:, None] * (last[:, None] - j).abs()[:, None]
    seen = (j <= last[:, None])[:, None]
    if state['layout'] is not None:
        seen = seen & state['layout'].transpose(0, 1)[last // block].repeat_interleave(block, 2)
    logits = logits.masked_fill(~seen, -math.inf)
    p = logits.sub_(logits.amax(-1, keepdim=True)).exp_()
    p = p.div_(p.sum(-1, keepdim=True))
    return torch.matmul(p, x[..., :latent].contiguous()).to(q.dtype)


def _run_expanded(state):
    case, q, k, v, qr, kr = state['case'], state['q'], state['k'], state['v'], state['qr'], state['kr']
    scale, cap, L = (case['dim'] + _SHARED) ** -0.5, case['softcap'], case['length']
    if own:
        rules = dict(scale=scale, softcap=cap, causal=case['causal'], documents=state['documents'], prefix=state['prefix'], shared=(qr, kr))
        if not case['train']:
            with torch.no_grad():
                return state['op'](q, k, v, **rules)
        o = state['op'](q, k, v, **rules)
        return (o.detach(),) + torch.autograd.grad(o, (q, k, v, qr, kr), state['do'])
    qf = torch.cat((q, qr), -1).float()
    kf = torch.cat((k, kr[:, None].expand(-1, k.size(1), -1, -1)), -1).float()
    vf = v.float()
    i = torch.arange(L, device='cuda')
    seen = state['layout'].repeat_interleave(case['block'], 1).repeat_interleave(case['block'], 2)[None, :, :L, :L]
    if case['causal']:
        visible = i[None, :] <= i[:, None]
        if state['prefix'] is not None:
            visible = visible | (i < state['prefix'][:, None, None, None])
        seen = seen & visible
    if state['documents'] is not None:
        ids = state['documents']
        seen = seen & ((ids[:, :, None] == ids[:, None, :]) & (ids[:, :, None] >= 0))[:, None]
    logits = torch.matmul(qf, kf.transpose(-1, -2)).mul_(scale)
    through = None
    if cap:
        logits = logits.div_(cap).tanh_()
        through = 1 - logits * logits if case['train'] else None
        logits = logits.mul_(cap)
    logits = logits.masked_fill_(~seen, -math.inf)
    most = logits.amax(-1, keepdim=True)
    p = logits.sub_(torch.where(most == -math.inf, 0., most)).exp_()
    total = p.sum(-1, keepdim=True)
    p = p.div_(torch.where(total == 0, 1., total))
    o = torch.matmul(p, vf)
    if not case['train']:
        return o.to(q.dtype)
    do = state['do'].float()
    dp = torch.matmul(do, vf.transpose(-1, -2))
    ds = dp.sub_((do * o).sum(-1, keepdim=True)).mul_(p)
    if cap:
        ds = ds.mul_(through)
    ds = ds.mul_(scale)
    d = case['dim']
    dq, dk = torch.matmul(ds, kf), torch.matmul(ds.transpose(-1, -2), qf)
    dv = torch.matmul(p.transpose(-1, -2), do)
    return tuple(x.to(q.dtype) for x in (o, dq[..., :d], dk[..., :d], dv, dq[..., d:], dk[..., d:].sum(1)))


# ---- what a pass cannot do without ---------------------------------------------------------------------------------------------------


def _visible(case):
    """pairs of a query and a key that it sees, over the batch and the heads"""
    Z, H, L, block = [case[n] for n in ('batch', 'heads', 'length', 'block')]
    blocks = (L + block - 1) // block
    layout = _layout(case['layout'], H, blocks, block, case['causal'] and not case['prefix'])
    ids = _documents(case) if case['documents'] else np.zeros((Z, L), np.int32)
    prefix = _prefix(case) if case['prefix'] else np.zeros(Z, np.int32)
    i = np.arange(L)
    row, alike = i // block, bool((layout == layout[:1]).all())
    total = 0
    for h in range(1 if alike else H):
        # keys of a block-row below a position: whole blocks before it, and what of its own block
        before = np.concatenate([np.zeros((blocks, 1), np.int64), np.cumsum(layout[h], 1) * block], 1)

        def below(end):
            full, rest = end // block, end % block
            return before[row, full] + np.where(rest > 0, layout[h][row, np.minimum(full, blocks - 1)] * rest, 0)

        for z in range(Z):
            order = ids[z] + (ids[z] < 0) * (1 << 30)
            lo, hi = np.searchsorted(order, ids[z]), np.searchsorted(order, ids[z], side='right')
            end = np.minimum(hi, np.maximum(i + 1, prefix[z])) if case['causal'] else hi
            n = np.where(ids[z] >= 0, np.maximum(below(end) - below(lo), 0), 0).sum()
            total += int(n) * (H if alike else 1)
    return total


def work(case):
    op, size = case['op'], _SIZE[case['dtype']]
    if op == 'rotate':
        n = case['batch'] * max(1, case['length']) * (case['heads'] + case['kv_heads'])
        passes = 2 if case['train'] else 1
        return dict(bytes=passes * 2 * n * case['dim'] * size + 4 * case['batch'] * max(1, case['length']), flops=passes * 3 * n * case['turned'])
    if op == 'append':
        T, H, d = case['tokens'], case['heads'], case['dim']
        if not H:
            return dict(bytes=T * (2 * (d + _SHARED) * size + 8), flops=3 * T * _SHARED)
        held = 2 * (d * case['bits'] // 8 + d // _GROUP * 4)          # a position of one head: key and value
        return dict(bytes=2 * T * H * (held + 2 * d * size) + 8 * T, flops=T * H * (8 * d + 3 * case['turned']))
    if op == 'latent':
        lengths, H, latent, block = _lengths(case), case['heads'], case['latent'], case['block']
        if case['layout'] == 'none':
            pairs, positions = int(lengths.sum()) * H, int(lengths.sum())
        else:
            layout = _layout(case['layout'], H, (case['length'] + block - 1) // block, block, True)
            pairs, positions = 0, 0
            for n in lengths:
                rows = layout[:, (n - 1) // block]                  # [H, block-columns]
                own_keys = np.clip(n - np.arange(rows.shape[1]) * block, 0, block)
                pairs += int((rows * own_keys).sum())
                positions += int((rows.any(0) * own_keys).sum())
        return dict(bytes=positions * (latent + _SHARED) * size + case['batch'] * H * (2 * latent + _SHARED) * size, flops=2 * (2 * latent + _SHARED) * pairs)
    Z, H, L, d, train = case['batch'], case['heads'], case['length'], case['dim'], case['train']
    q, r, kr = [Z * n * L * size for n in (H * d, H * _SHARED, _SHARED)]       # q, k, v and o are of one size here
    pairs = _visible(case)
    return dict(bytes=(8 * q + 2 * r + 2 * kr) if train else 4 * q + r + kr, flops=((12 * d + 6 * _SHARED) if train else 4 * d + 2 * _SHARED) * pairs)


# ---- in 64 bits -------------------------------------------------------------------------------------------------------------------


def _sixty_four(x, bits):
    """a key or value as the cache holds it, from the definition: of 32 values the least, rounded to fp16, and the rest in steps of
    (greatest - least) / (2^bits - 1), rounded to fp16"""
    x = torch.clamp(x.to(torch.float64), -65504., 65504.)
    g = x.reshape(x.shape[:-1] + (x.shape[-1] // _GROUP, _GROUP))
    least = g.min(-1, keepdim=True).values.to(torch.float16).to(torch.float64)
    step = ((g.max(-1, keepdim=True).values - least) / float(2 ** bits - 1)).to(torch.float16).to(torch.float64)
    n = torch.clamp(torch.round((g - least) / step), 0, 2 ** bits - 1)
    n[(step == 0).expand_as(n)] = 0
    return (least + n * step).reshape(x.shape)


def _complex_turn(case, x, positions, sign=1.):
    """the same turn as a product of complex numbers; positions broadcast against x without its last dimension"""
    n = case['turned'] // 2
    omega = torch.exp(-math.log(case['base']) * torch.arange(n, dtype=torch.float64, device='cuda') / n)
    by = torch.polar(torch.ones((), dtype=torch.float64, device='cuda'), sign * positions.to(torch.float64)[..., None] * omega)
    x = x.detach().to(torch.float64)
    out = x.clone()
    first, second = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if case['neighbours'] else (slice(0, n), slice(n, 2 * n))
    z = torch.complex(x[..., first].contiguous(), x[..., second].contiguous()) * by
    out[..., first], out[..., second] = z.real, z.imag
    return out


def exact(case, seed):
    x = _inputs(case, seed)
    if case['op'] == 'rotate':
        positions = x['positions'][:, None]
        out = [_complex_turn(case, x[n], positions) for n in ('q', 'k')]
        return tuple(out + ([_complex_turn(case, x[n], positions, -1.) for n in ('dq', 'dk')] if case['train'] else []))
    if case['op'] == 'append':
        if case['heads']:
            return _sixty_four(_complex_turn(case, x['k'], x['positions'][:, None]), case['bits']), _sixty_four(x['v'], case['bits'])
        pages = torch.zeros(x['pages'] * case['block'], case['dim'] + _SHARED, dtype=torch.float64, device='cuda')
        pages[x['slots'].long(), :case['dim']] = x['c'].double()
        pages[x['slots'].long(), case['dim']:] = _complex_turn(case, x['r'], x['positions'])
        return pages.view(x['pages'], case['block'], -1)
    return _exact_latent(case, x) if case['op'] == 'latent' else _exact_expanded(case, x)


def _exact_latent(case, x):
    H, block, latent = case['heads'], case['block'], case['latent']
    layout = None if case['layout'] == 'none' else torch.from_numpy(_layout(case['layout'], H, x['table'].size(1), block, True)).cuda()
    slopes = _slopes(H).double().cuda()
    out = torch.empty(case['batch'], H, latent, dtype=torch.float64, device='cuda')
    for b, n in enumerate(_lengths(case).tolist()):
        where = (x['table'][b].long()[:, None] * block + torch.arange(block, device='cuda')).reshape(-1)[:n]
        c, r = x['c'][where].double(), x['r'][where].double()
        s = (x['q'][b].double() @ c.T + x['qr'][b].double() @ r.T) / math.sqrt(128 + _SHARED)
        if case['softcap']:
            s = case['softcap'] * torch.tanh(s / case['softcap'])
        if case['slopes']:
            s = s - slopes[:, None] * torch.arange(n - 1, -1, -1, device='cuda', dtype=torch.float64)
        if layout is not None:
            s = s.masked_fill(~layout[:, (n - 1) // block].repeat_interleave(block, 1)[:, :n], -math.inf)
        w = torch.exp(s - s.max(1, keepdim=True).values)
        out[b] = (w @ c) / w.sum(1, keepdim=True)
    return out


def _exact_expanded(case, x):
    q, k, v, qr, kr = [x[n].double() for n in ('q', 'k', 'v', 'qr', 'kr')]
    Z, H, L, d, block, cap = [case[n] for n in ('batch', 'heads', 'length', 'dim', 'block', 'softcap')]
    layout = _layout(case['layout'], H, (L + block - 1) // block, block, case['causal'] and not case['prefix'])
    o, dq, dk, dv, dqr, dkr = [torch.zeros_like(t) for t in (v, q, k, v, qr, kr)]
    pos = torch.arange(L, device='cuda')
    scale = 1. / math.sqrt(d + _SHARED)
    for z in range(Z):
        rule = torch.ones(L, L, dtype=torch.bool, device='cuda')
        if case['causal']:
            rule = pos[:, None] >= pos[None, :]
            if case['prefix']:
                rule = rule | (pos < int(_prefix(case)[z]))[None, :]
        if case['documents']:
            ids = torch.from_numpy(_documents(case)[z]).cuda()
            rule = rule & (ids[:, None] == ids[None, :]) & (ids >= 0)[None, :]
        for h in range(H):
            see = rule & torch.from_numpy(layout[h]).cuda().repeat_interleave(block, 0).repeat_interleave(block, 1)[:L, :L]
            s = (q[z, h] @ k[z, h].T + qr[z, h] @ kr[z].T) * scale
            t = torch.tanh(s / cap) if cap else None
            y = torch.where(see, cap * t if cap else s, -math.inf)
            w = torch.exp(y - y.max(1, keepdim=True).values.clamp(min=-1e300))
            w = w / w.sum(1, keepdim=True).clamp(min=1e-300)
            o[z, h] = w @ v[z, h]
            if case['train']:
                do = x['do'][z, h].double()
                dv[z, h] = w.T @ do
                e = do @ v[z, h].T
                e = w * (e - (w * e).sum(1, keepdim=True)) * scale
                if cap:
                    e = e * (1 - t * t)
                dq[z, h], dk[z, h] = e @ k[z, h], e.T @ q[z, h]
                dqr[z, h] = e @ kr[z]
                dkr[z] += e.T @ qr[z, h]
    return (o, dq, dk, dv, dqr, dkr) if case['train'] else o
