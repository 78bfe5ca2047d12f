"""The dense operators around the sparse products, as a user calls them: embedding lookup, residual RMS norm (training, and with an
8-bit output for serving), the gated feed-forward product, and the 8-bit matrix product with a scale for each block of 128.

``listed()`` names the cases, ``prepare`` makes a case's inputs, ``run`` makes one pass: with ``own`` through ``dgsparse``, without
it in elementary torch operations in 32 bits.  ``exact`` is the same result from the definition in 64 bits.

Definitions (x row-major, one token or graph node a row):

  embedding   out[p] = scale * table[ids[p]]; a negative id stands for "no token": its row is 0 and it adds to no gradient
              dtable[v] = scale * sum over p with ids[p] = v of dout[p]
  norm        s = x + residual, rounded to x's type (it is the residual that the next layer reads); y = s / sqrt(mean(s^2) + eps) * w
              dx = dresidual = r (w dy) - s r^3 mean(s w dy) + ds with r = 1 / sqrt(mean(s^2) + eps);  dw = sum over rows of dy s r
  norm8       the same y, given as 8-bit floating point (e4m3): per row and block of 128 columns scale = max|y| / 448, q = y / scale
  ffn         h = act(x Wg^T) * (x Wu^T)  with Wg, Wu [F, D];  with g, u the two products: dg = dh u act'(g), du = dh act(g),
              dx = dg Wg + du Wu, dWg = dg^T x, dWu = du^T x
  mm8         out = A B^T, A [M, K] in e4m3 with a scale for each row and block of 128 columns, B [N, K] with a scale for each block of
              128 x 128
"""
import math
import os
import sys

import torch

own = False

EPS = 1e-6
BLOCK = 128     # columns (and, for weights, rows) that share a scale
E4M3_MAX = 448.0
TYPES = {'fp32': torch.float32, 'fp16': torch.float16, 'bf16': torch.bfloat16}


def _api():
    """The framework (imported only where `own` is true)."""
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), 'dgsparse-lib_amd')
    if root not in sys.path:
        sys.path.insert(0, root)
    import dgsparse
    return dgsparse


# ---- the cases --------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # one step of 33 sequences that are being answered: the lookup alone, latency counts
        dict(name='embed_decode', op='embedding', train=False, n=33, vocab=32000, dim=4096, dtype='fp16', padded=0.0, scale=64.0),
        # a training batch of 16 sequences of 1024 tokens, Zipf-distributed, some positions padded; the gradient is the whole table's
        dict(name='embed_tokens', op='embedding', train=True, n=16384, vocab=131072, dim=4096, dtype='bf16', padded=0.04, scale=1.0),
        # node embeddings of an arxiv-sized graph, looked up for the rows of a sampled neighbourhood (hubs come up again and again)
        dict(name='embed_nodes', op='embedding', train=True, n=100003, vocab=169343, dim=128, dtype='fp32', padded=0.0, scale=1.0),
        # a residual layer of a graph network over all nodes of an arxiv-sized graph
        dict(name='norm_nodes', op='norm', train=True, rows=169343, dim=128, dtype='fp32'),
        # a residual layer over a training batch of tokens
        dict(name='norm_tokens', op='norm', train=True, rows=8192, dim=4096, dtype='bf16'),
        # the same layer in serving, in front of an 8-bit product: one step of seven sequences, then a long prompt
        dict(name='norm8_decode', op='norm8', rows=7, dim=4096, dtype='bf16'),
        dict(name='norm8_prompt', op='norm8', rows=8191, dim=5120, dtype='fp16'),
        # the update function of a graph layer over all nodes: many rows, a narrow product
        dict(name='ffn_nodes', op='ffn', train=True, rows=169343, dim=128, hidden=512, dtype='fp32', act='gelu'),
        # the feed-forward block of a training batch
        dict(name='ffn_tokens', op='ffn', train=True, rows=4096, dim=4096, hidden=11008, dtype='bf16', act='silu'),
        # ... and of one step of three sequences that are being answered
        dict(name='ffn_decode', op='ffn', train=False, rows=3, dim=2048, hidden=5504, dtype='fp16', act='silu'),
        # the projection behind it in 8 bits: one step of five sequences, then a long prompt
        dict(name='mm8_decode', op='mm8', rows=5, cols=4096, inner=11008, dtype='bf16'),
        dict(name='mm8_prompt', op='mm8', rows=4095, cols=11000, inner=4096, dtype='bf16'),
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _width(rng, lo, hi):
    """A row width: mostly a multiple of 64 or 8, one in four odd."""
    n = _log(rng, lo, hi)
    step = rng.choice((64, 64, 8, 1))
    return max(lo, n // step * step)


def draw(rng):
    op = rng.choice(('embedding', 'embedding', 'norm', 'norm8', 'ffn', 'ffn', 'mm8', 'mm8'))
    dtype = rng.choice(('fp32', 'fp16', 'bf16'))
    if op == 'embedding':
        train = rng.random() < 0.7
        dim = _width(rng, 16, 4096)
        return dict(op=op, train=train, n=_log(rng, 1, min(100003, (1 << 26) // dim)), vocab=_log(rng, 500, min(169343, (1 << 29) // dim)), dim=dim,
                    dtype=dtype, padded=rng.choice((0.0, 0.0, 0.1, 0.5)), scale=rng.choice((1.0, 0.5, 8.0)))
    if op == 'norm':
        dim = _width(rng, 32, 8192)
        return dict(op=op, train=True, rows=_log(rng, 1, min(169343, (1 << 25) // dim)), dim=dim, dtype=dtype)
    if op == 'norm8':
        dim = _width(rng, 64, 8192)
        return dict(op=op, rows=_log(rng, 1, min(169343, (1 << 25) // dim)), dim=dim, dtype=rng.choice(('fp16', 'bf16')))
    if op == 'ffn':
        train = rng.random() < 0.6
        dim = _width(rng, 32, 4096)
        hidden = _width(rng, 64, 11008)
        most = int(2e11 if dtype == 'fp32' else 1e12) // (12 * dim * hidden)
        if not train:
            most = min(most, rng.choice((64, 16384)))
        return dict(op=op, train=train, rows=_log(rng, 1, max(1, min(169343, most))), dim=dim, hidden=hidden, dtype=dtype,
                    act=rng.choice(('silu', 'gelu') if dtype == 'fp32' else ('silu', 'gelu', 'relu')))  # (relu': 32 bits cannot say on which side of 0)
    inner, cols = _width(rng, 128, 11008), _width(rng, 128, 11008)
    return dict(op=op, rows=_log(rng, 1, max(1, min(16384, int(3e11) // (2 * inner * cols)))), cols=cols, inner=inner,
                dtype=rng.choice(('fp16', 'bf16', 'fp32')))


# ---- inputs -----------------------------------------------------------------------------------------------------------------
def _quantised(x, rows):
    """(e4m3 values, scales) of x with one scale for each `rows` x 128 values: how a checkpoint in 8 bits is laid out."""
    m, k = x.shape
    bm, bk = -(-m // rows), -(-k // BLOCK)
    padded = torch.zeros(bm * rows, bk * BLOCK, device=x.device)
    padded[:m, :k] = x
    tiles = padded.view(bm, rows, bk, BLOCK)
    scale = tiles.abs().amax(dim=(1, 3)).clamp_min(2.0 ** -96) / E4M3_MAX
    q = (tiles / scale[:, None, :, None]).view(bm * rows, bk * BLOCK)[:m, :k].contiguous()
    return q.to(torch.float8_e4m3fn), scale.contiguous()


def prepare(case, seed):
    g = torch.Generator(device='cuda').manual_seed(seed)

    def normal(*shape, scale=1.0, dtype=torch.float32):
        return (torch.randn(*shape, generator=g, device='cuda') * scale).to(dtype)

    op, t = case['op'], TYPES[case['dtype']]
    state = dict(case=case)
    if op == 'embedding':
        n, vocab, dim = case['n'], case['vocab'], case['dim']
        # Zipf's law with exponent 1 over a shuffled vocabulary
        rank = torch.rand(n, generator=g, device='cuda', dtype=torch.float64).mul(math.log(vocab + 1)).exp().long().sub(1).clamp(0, vocab - 1)
        ids = torch.randperm(vocab, generator=g, device='cuda')[rank]
        ids = torch.where(torch.rand(n, generator=g, device='cuda') < case['padded'], torch.full_like(ids, -1), ids)
        state.update(ids=ids, table=normal(vocab, dim, scale=0.02, dtype=t), scale=case['scale'])
        if case['train']:
            state.update(dout=normal(n, dim, dtype=t))
            state['table'].requires_grad_()
    elif op in ('norm', 'norm8'):
        rows, dim = case['rows'], case['dim']
        state.update(x=normal(rows, dim, dtype=t), residual=normal(rows, dim, scale=3.0, dtype=t),
                     weight=(1.0 + 0.1 * normal(dim)).to(t))
        if op == 'norm':
            state.update(dy=normal(rows, dim, dtype=t), ds=normal(rows, dim, dtype=t))
            for k in ('x', 'residual', 'weight'):
                state[k].requires_grad_()
    elif op == 'ffn':
        rows, dim, hidden = case['rows'], case['dim'], case['hidden']
        state.update(x=normal(rows, dim, dtype=t), w_gate=normal(hidden, dim, scale=dim ** -0.5, dtype=t),
                     w_up=normal(hidden, dim, scale=dim ** -0.5, dtype=t))
        if case['train']:
            state.update(dh=normal(rows, hidden, dtype=t))
            for k in ('x', 'w_gate', 'w_up'):
                state[k].requires_grad_()
    else:
        rows, cols, inner = case['rows'], case['cols'], case['inner']
        a, a_scale = _quantised(normal(rows, inner), 1)
        b, b_scale = _quantised(normal(cols, inner, scale=inner ** -0.5), BLOCK)
        state.update(a=a, a_scale=a_scale, b=b, b_scale=b_scale)
    return state


# ---- one pass ---------------------------------------------------------------------------------------------------------------
def _act(name, g):
    """act(g) and act'(g)."""
    if name == 'relu':
        return torch.clamp(g, min=0.0), (g > 0).to(g.dtype)
    if name == 'silu':
        sig = 1.0 / (1.0 + torch.exp(-g))
        return g * sig, sig * (1.0 + g * (1.0 - sig))
    cdf = 0.5 * (1.0 + torch.erf(g * math.sqrt(0.5)))
    return g * cdf, cdf + g * torch.exp(-0.5 * g * g) * (1.0 / math.sqrt(2.0 * math.pi))


def _plain_embedding(s):
    table, ids, t = s['table'].detach(), s['ids'], s['table'].dtype
    there = ids >= 0
    rows = table[ids.clamp_min(0)].float() * s['scale']
    out = torch.where(there[:, None], rows, torch.zeros_like(rows)).to(t)
    if not s['case']['train']:
        return out
    grad = torch.zeros(table.shape, dtype=torch.float32, device=table.device)
    grad.index_add_(0, ids.clamp_min(0), torch.where(there[:, None], s['dout'].float(), torch.zeros_like(rows)))
    return dict(out=out, dtable=(grad * s['scale']).to(t))


def _plain_norm(s):
    x, t = s['x'].detach(), s['x'].dtype
    new = (x.float() + s['residual'].detach().float()).to(t)
    v, w = new.float(), s['weight'].detach().float()
    r = torch.rsqrt((v * v).mean(dim=1, keepdim=True) + EPS)
    y = v * r * w
    if s['case']['op'] == 'norm8':
        rows, dim = y.shape
        blocks = -(-dim // BLOCK)
        tiles = torch.nn.functional.pad(y, (0, blocks * BLOCK - dim)).view(rows, blocks, BLOCK)
        scale = tiles.abs().amax(dim=2).clamp_min(2.0 ** -96) / E4M3_MAX
        q = (tiles / scale[:, :, None]).view(rows, blocks * BLOCK)[:, :dim]
        return dict(q=q.to(torch.float8_e4m3fn), scale=scale, residual=new)
    dy, ds = s['dy'].float(), s['ds'].float()
    wdy = w * dy
    dv = r * wdy - v * r * r * r * (v * wdy).mean(dim=1, keepdim=True) + ds
    return dict(y=y.to(t), residual=new, dx=dv.to(t), dresidual=dv.to(t), dweight=(dy * v * r).sum(dim=0).to(t))


def _plain_ffn(s):
    t = s['x'].dtype
    x, wg, wu = s['x'].detach().float(), s['w_gate'].detach().float(), s['w_up'].detach().float()
    g, u = x @ wg.t(), x @ wu.t()
    a, da = _act(s['case']['act'], g)
    h = (a * u).to(t)
    if not s['case']['train']:
        return h
    dh = s['dh'].float()
    dg, du = dh * u * da, dh * a
    return dict(h=h, dx=(dg @ wg + du @ wu).to(t), dw_gate=(dg.t() @ x).to(t), dw_up=(du.t() @ x).to(t))


def _plain_mm8(s):
    k, n = s['a'].shape[1], s['b'].shape[0]
    a = s['a'].float() * s['a_scale'].repeat_interleave(BLOCK, dim=1)[:, :k]
    b = s['b'].float() * s['b_scale'].repeat_interleave(BLOCK, dim=0)[:n].repeat_interleave(BLOCK, dim=1)[:, :k]
    return (a @ b.t()).to(TYPES[s['case']['dtype']])


def run(state):
    case = state['case']
    op = case['op']
    if own:
        dgsparse = _api()
        if op == 'embedding':
            out = dgsparse.embedding(state['ids'], state['table'], scale=state['scale'])
            if not case['train']:
                return out
            dtable, = torch.autograd.grad(out, state['table'], state['dout'])
            return dict(out=out, dtable=dtable)
        if op == 'norm':
            y, new = dgsparse.add_rms_norm(state['x'], state['residual'], state['weight'], EPS)
            dx, dres, dw = torch.autograd.grad((y, new), (state['x'], state['residual'], state['weight']), (state['dy'], state['ds']))
            return dict(y=y, residual=new, dx=dx, dresidual=dres, dweight=dw)
        if op == 'norm8':
            q, scale, new = dgsparse.add_rms_norm_fp8(state['x'], state['residual'], state['weight'], EPS)
            return dict(q=q, scale=scale, residual=new)
        if op == 'ffn':
            h = dgsparse.gated_ffn(state['x'], state['w_gate'], state['w_up'], case['act'])
            if not case['train']:
                return h
            dx, dwg, dwu = torch.autograd.grad(h, (state['x'], state['w_gate'], state['w_up']), state['dh'])
            return dict(h=h, dx=dx, dw_gate=dwg, dw_up=dwu)
        return dgsparse.matmul_fp8(state['a'], state['a_scale'], state['b'], state['b_scale'], TYPES[case['dtype']])
    if op == 'embedding':
        return _plain_embedding(state)
    if op in ('norm', 'norm8'):
        return _plain_norm(state)
    if op == 'ffn':
        return _plain_ffn(state)
    return _plain_mm8(state)


# ---- what a pass cannot do without ------------------------------------------------------------------------------------------
def work(case):
    op, size = case['op'], TYPES[case['dtype']].itemsize
    if op == 'embedding':
        n, dim, vocab = case['n'], case['dim'], case['vocab']
        found = n * (1.0 - case['padded'])
        moved = n * 8 + (found + n) * dim * size                         # ids, the rows, the output
        if case['train']:
            moved += n * 8 + found * dim * size + vocab * dim * size     # ids, the output's gradient, the whole table's gradient
        return dict(bytes=moved, flops=found * dim * (2 if case['train'] else 1))
    if op in ('norm', 'norm8'):
        rows, dim = case['rows'], case['dim']
        if op == 'norm8':
            return dict(bytes=rows * (3 * dim * size + dim + 4 * -(-dim // BLOCK)) + dim * size, flops=8 * rows * dim)
        # forward: x, residual -> s, y; backward: dy, ds, s -> the one gradient that x and the residual share
        return dict(bytes=8 * rows * dim * size + 3 * dim * size, flops=16 * rows * dim)
    if op == 'ffn':
        rows, dim, hidden = case['rows'], case['dim'], case['hidden']
        moved, flops = rows * dim + 2 * hidden * dim + rows * hidden, 4 * rows * dim * hidden  # x, the weights, h
        if case['train']:                                                                      # ... dh, dx and the weights' gradients
            moved, flops = 2 * moved, 3 * flops
        return dict(bytes=moved * size, flops=flops)
    rows, cols, inner = case['rows'], case['cols'], case['inner']
    blocks = -(-inner // BLOCK)
    return dict(bytes=rows * inner + cols * inner + 4 * blocks * (rows + -(-cols // BLOCK)) + rows * cols * size, flops=2 * rows * cols * inner)


# ---- the definition in 64 bits ----------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    op = case['op']
    with torch.enable_grad():
        if op == 'embedding':
            kept = (s['ids'] >= 0).nonzero().flatten()
            ids = s['ids'][kept]
            out = torch.zeros(case['n'], case['dim'], dtype=torch.float64, device='cuda')
            out[kept] = s['table'].detach().double().index_select(0, ids) * s['scale']
            if not case['train']:
                return out
            grad = torch.zeros(case['vocab'], case['dim'], dtype=torch.float64, device='cuda')
            grad.index_put_((ids,), s['dout'][kept].double() * s['scale'], accumulate=True)
            return dict(out=out, dtable=grad)
        if op in ('norm', 'norm8'):
            new = (s['x'].detach().double() + s['residual'].detach().double()).to(s['x'].dtype)
            v = new.double().requires_grad_()
            w = s['weight'].detach().double().requires_grad_()
            y = v / torch.sqrt(v.square().sum(1, keepdim=True) / case['dim'] + EPS) * w
            if op == 'norm8':
                y = y.detach()
                parts = [y[:, c:c + BLOCK] for c in range(0, case['dim'], BLOCK)]
                scales = [p.abs().max(dim=1).values.clamp_min(2.0 ** -96) / E4M3_MAX for p in parts]
                return dict(q=torch.cat([p / c[:, None] for p, c in zip(parts, scales)], dim=1), scale=torch.stack(scales, dim=1), residual=new.double())
            dv, dw = torch.autograd.grad((y, v * 1.0), (v, w), (s['dy'].double(), s['ds'].double()))
            return dict(y=y.detach(), residual=new.double(), dx=dv, dresidual=dv, dweight=dw)
        if op == 'ffn':
            x, wg, wu = (s[k].detach().double().requires_grad_() for k in ('x', 'w_gate', 'w_up'))
            act = dict(relu=torch.nn.functional.relu, silu=torch.nn.functional.silu, gelu=torch.nn.functional.gelu)[case['act']]
            h = act(torch.nn.functional.linear(x, wg)) * torch.nn.functional.linear(x, wu)
            if not case['train']:
                return h.detach()
            dx, dwg, dwu = torch.autograd.grad(h, (x, wg, wu), s['dh'].double())
            return dict(h=h.detach(), dx=dx, dw_gate=dwg, dw_up=dwu)
        out = torch.zeros(case['rows'], case['cols'], dtype=torch.float64, device='cuda')
        for b, c in enumerate(range(0, case['inner'], BLOCK)):
            part = s['a'][:, c:c + BLOCK].double() @ s['b'][:, c:c + BLOCK].double().t()
            per_col = s['b_scale'][:, b].double()[torch.arange(case['cols'], device='cuda') // BLOCK]
            out += part * s['a_scale'][:, b].double()[:, None] * per_col[None, :]
        return out
