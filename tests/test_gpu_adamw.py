"""The many-tensor optimizer step (unetk.optim.AdamW, clip_grad_norm_) against its 64-bit restatement, element by element, with
tolerances counted from the roundings that fp32 arithmetic makes (oracle/adamw_np.py)."""
import copy
import math

import numpy as np
import pytest
import torch

from oracle import adamw_np as O

pytestmark = pytest.mark.gpu

HYPER = dict(lr=1e-2, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.1)
TYPES = {'fp32': torch.float32, 'bf16': torch.bfloat16, 'fp16': torch.float16}
COEF_ERR = 6 * O.U                    # of the norm (2), the sum with 1e-6, the quotient, the product with the scale's inverse


@pytest.fixture(scope='module')
def optim():
    from unetk import optim
    return optim


def f64(t):
    return t.detach().double().cpu().numpy().ravel()


def mem(t):
    """A dense tensor's values in memory order."""
    return f64(t.as_strided((t.numel(),), (1,)))


def make(sizes, dtype, seed=0, scale=1e-2):
    g = torch.Generator().manual_seed(seed)
    out = []
    for n in sizes:
        p = torch.nn.Parameter((torch.randn(n, generator=g) * 0.1).to(dtype).cuda())
        p.grad = (torch.randn(n, generator=g) * scale * 10 ** (2 * torch.rand((), generator=g) - 1)).to(dtype).cuda()
        out.append(p)
    return out


def snapshot(opt, params):
    rec = []
    for p in params:
        st = opt.state.get(p) or {}
        r = dict(p=mem(p), g=None if p.grad is None else mem(p.grad), t=float(st['step']) if st else 0.0)
        n = p.numel()
        if 'scales' in st:
            k = st['scales'].view(torch.uint8).cpu().numpy().astype(int) - 127
            r['k'] = (k[:, 0], k[:, 1])
            r['codes'] = (mem(st['exp_avg'].float()), mem(st['exp_avg_root'].float()))
            r['m'], root = (np.ldexp(c, np.repeat(kk, 256)[:n]) for c, kk in zip(r['codes'], r['k']))
            r['v'] = root ** 2
        elif st:
            r['m'], r['v'] = mem(st['exp_avg']), mem(st['exp_avg_sq'])
        else:
            r['m'] = r['v'] = np.zeros(n)
        rec.append(r)
    return rec


def check_step(params, before, after, hyper, max_norm=None, seed=0, total_norm=None, norm=None):
    factor, err = 1.0, 0.0
    if max_norm is not None:
        norm = O.norm([b['g'] for b in before if b['g'] is not None]) if norm is None else norm
        assert abs(float(total_norm) - norm) <= 3 * O.U * norm
        factor, err = O.clip_coef(norm, max_norm), COEF_ERR
    for p, b, a in zip(params, before, after):
        if b['g'] is None:
            assert a['t'] == b['t'] and np.array_equal(a['p'], b['p'])
            continue
        t = b['t'] + 1
        assert a['t'] == t
        fi = torch.finfo(p.dtype)
        half, tiny = (0.0, 0.0) if p.dtype == torch.float32 else (fi.eps / 2, fi.smallest_normal)
        want = O.step(b['p'], b['g'], b['m'], b['v'], t, hyper['lr'], *hyper['betas'], hyper['eps'], hyper['weight_decay'],
                      factor, err, half, tiny)
        assert (np.abs(a['p'] - want['p']) <= want['pe']).all(), np.abs(a['p'] - want['p']).max()
        if 'k' not in a:
            assert (np.abs(a['m'] - want['m']) <= want['me']).all()
            assert (np.abs(a['v'] - want['v']) <= want['ve']).all()
            continue
        for x, xe, k, codes, u, root in zip((want['m'], want['r']), (want['me'], want['re']), a['k'], a['codes'],
                                            O.fractions(len(b['p']), t, seed), (False, True)):
            for kk, lo, hi in zip(k, O.scale_exponent(np.maximum(np.abs(x) - xe, 0)), O.scale_exponent(np.abs(x) + xe)):
                assert lo <= kk <= hi
            lo, hi = O.code_range(x, xe, k, u, root)
            assert (lo <= codes).all() and (codes <= hi).all()
            # the bound leaves a choice at almost no element -- but where a square falls among fp32's subnormals, whose root may
            # be off by 2^-74 and so be anything among the smallest
            clear = xe <= 1e-6 * np.abs(x)
            assert clear.sum() < 1000 or (lo == hi)[clear].mean() > 0.99


SIZES = {'one': [1], 'small': [3, 1, 2, 255, 256, 257], 'edges': [4095, 4096, 4097, 8191, 12288 + 1], 'mixed': [100003, 7, 4096, 65537, 64],
         'many': [1 + (37 * i) % 700 for i in range(64)], 'more': [1 + (53 * i) % 500 for i in range(65)],
         'lots': [1 + (29 * i) % 300 for i in range(200)], 'most': [(31 * i) % 90 for i in range(385)] + [9001]}


@pytest.mark.parametrize('sizes', list(SIZES))
@pytest.mark.parametrize('bits', [32, 8])
@pytest.mark.parametrize('dtype', list(TYPES))
@pytest.mark.parametrize('max_norm', [None, 0.5])
def test_steps(optim, sizes, bits, dtype, max_norm):
    params = make(SIZES[sizes], TYPES[dtype], seed=len(sizes))
    opt = optim.AdamW(params, **HYPER, max_norm=max_norm, state_bits=bits, min_8bit_numel=1, seed=77)
    for k in range(3):
        before = snapshot(opt, params)
        opt.step()
        after = snapshot(opt, params)
        check_step(params, before, after, HYPER, max_norm, 77, opt.total_norm)
        assert all(np.array_equal(b['g'], a['g']) for a, b in zip(after, before))      # gradients stay as they are
        for i, p in enumerate(params):
            p.grad = torch.randn_like(p) * 10.0 ** (-2 - (i + k) % 3)


@pytest.mark.parametrize('bits', [32, 8])
def test_no_limit_reached_and_extreme_hyperparameters(optim, bits):
    """A limit above the norm changes nothing; beta 0, weight decay 0, eps 0 and lr 0 are what the formula says."""
    for hyper, max_norm in ((HYPER, 1e6), (dict(lr=1e-3, betas=(0.0, 0.9), eps=1e-3, weight_decay=0.0), 1e6),
                            (dict(lr=0.0, betas=(0.9, 0.0), eps=1e-8, weight_decay=0.0), None)):
        a, b = make([5000, 33], torch.float32), make([5000, 33], torch.float32)
        oa = optim.AdamW(a, **hyper, max_norm=max_norm, state_bits=bits, min_8bit_numel=1)
        ob = optim.AdamW(b, **hyper, state_bits=bits, min_8bit_numel=1)
        for _ in range(2):
            before = snapshot(oa, a)
            oa.step(), ob.step()
            check_step(a, before, snapshot(oa, a), hyper, max_norm, 0, oa.total_norm)
        assert all(torch.equal(x, y) for x, y in zip(a, b))
        if hyper['lr'] == 0.0:
            assert all(torch.equal(x, y) for x, y in zip(a, make([5000, 33], torch.float32)))


@pytest.mark.parametrize('bits', [32, 8])
def test_groups_and_types_side_by_side(optim, bits):
    """One norm over every group and type, each group's own hyperparameters; a scheduler moves one of them."""
    fp32, bf16, fp16 = make([5000, 30], torch.float32), make([4500, 7, 0], torch.bfloat16, 1), make([9000], torch.float16, 2)
    opt = optim.AdamW([{'params': fp32 + bf16, 'lr': 1e-2}, {'params': fp16, 'lr': 1e-3, 'betas': (0.5, 0.95), 'weight_decay': 0.0}],
                      max_norm=0.2, state_bits=bits, seed=1)
    sched = torch.optim.lr_scheduler.LambdaLR(opt, [lambda k: 1.0, lambda k: 0.5 ** k])
    params = fp32 + bf16 + fp16
    for k in range(3):
        before = snapshot(opt, params)
        opt.step()
        after = snapshot(opt, params)
        norm = O.norm([b['g'] for b in before])
        assert abs(float(opt.total_norm) - norm) <= 3 * O.U * norm
        # each group against its own formula, under the common factor
        for lo, hi, hyper in ((0, 5, dict(HYPER, betas=(0.9, 0.999), weight_decay=1e-2)),
                              (5, 6, dict(lr=1e-3 * 0.5 ** k, betas=(0.5, 0.95), eps=1e-8, weight_decay=0.0))):
            check_step(params[lo:hi], before[lo:hi], after[lo:hi], hyper, 0.2, 1, opt.total_norm, norm=norm)
        sched.step()


def test_nothing_but_empty_tensors(optim):
    params = make([0, 0], torch.float32)
    opt = optim.AdamW(params, max_norm=1.0)
    opt.step()
    assert float(opt.total_norm) == 0.0 and float(opt.state[params[0]]['step']) == 1.0
    assert float(optim.clip_grad_norm_(params, 1.0)) == 0.0


def test_the_norm_of_no_gradients_is_zero(optim):
    params = make([50, 5000], torch.float32)
    opt = optim.AdamW(params, max_norm=1.0)
    opt.step()
    assert float(opt.total_norm) > 0
    opt.zero_grad()
    opt.step()
    assert opt.total_norm.is_cuda and opt.total_norm.dtype == torch.float32 and float(opt.total_norm) == 0.0
    opt.param_groups[0]['max_norm'] = None
    opt.step()
    assert opt.total_norm is None


@pytest.mark.parametrize('dtype', list(TYPES))
@pytest.mark.parametrize('bits', [32, 8])
@pytest.mark.parametrize('shift', [1, 3])
def test_views_at_any_address_touch_nothing_else(optim, dtype, bits, shift):
    """Tensors that lie one behind the other at odd elements of one buffer, with a guard in front, between and behind."""
    dt, sizes, gap = TYPES[dtype], [1, 257, 4096, 4099, 31, 70001], 5
    off, starts = shift, []
    for n in sizes:
        starts.append(off)
        off += n + gap
    g = torch.Generator().manual_seed(1)

    def buffer(d):
        raw = torch.randn(off + 8, generator=g).cuda()
        return raw.to(d) if d.itemsize > 1 else (raw.abs() * 8).to(d)

    bufs = {k: buffer(d) for k, d in (('p', dt), ('g', dt), ('m', torch.float32 if bits == 32 else torch.float8_e4m3fn),
                                      ('v', torch.float32 if bits == 32 else torch.float8_e4m3fn))}
    if bits == 32:
        bufs['v'].abs_()
    saved = {k: v.clone() for k, v in bufs.items()}
    views = {k: [b[a:a + n] for a, n in zip(starts, sizes)] for k, b in bufs.items()}
    params = [torch.nn.Parameter(p) for p in views['p']]
    opt = optim.AdamW(params, **HYPER, max_norm=1.0, state_bits=bits, min_8bit_numel=1)
    for i, (p, n) in enumerate(zip(params, sizes)):
        p.grad = views['g'][i]
        opt.state[p] = {'step': torch.full((), 4.0, device='cuda'), 'exp_avg': views['m'][i],
                        ('exp_avg_sq' if bits == 32 else 'exp_avg_root'): views['v'][i]}
        if bits == 8:
            scales = torch.full((2 * -(-n // 256) + 1,), 125, dtype=torch.uint8, device='cuda')[i % 2:][:2 * -(-n // 256)]
            opt.state[p]['scales'] = scales.view(-1, 2).view(torch.float8_e8m0fnu)          # at an odd address, too
    before = snapshot(opt, params)
    opt.step()
    check_step(params, before, snapshot(opt, params), HYPER, 1.0, 0, opt.total_norm)
    inside = torch.zeros(off + 8, dtype=torch.bool)
    for a, n in zip(starts, sizes):
        inside[a:a + n] = True
    for k, b in bufs.items():
        raw = torch.uint8 if b.element_size() == 1 else torch.int16 if b.element_size() == 2 else torch.int32
        same = (b.view(raw) == saved[k].view(raw)).cpu()
        assert same[~inside].all(), k
        assert k != 'g' or same.all()


def test_empty_tensors_missing_gradients_and_own_step_counts(optim):
    params = make([10, 0, 5000, 7, 0], torch.float32)
    opt = optim.AdamW(params, **HYPER, max_norm=1.0, state_bits=8)
    for k in range(4):
        params[2].grad = None if k == 1 else torch.randn_like(params[2])
        before = snapshot(opt, params)
        opt.step()
        check_step(params, before, snapshot(opt, params), HYPER, 1.0, 0, opt.total_norm)
    assert float(opt.state[params[2]]['step']) == 3.0 and float(opt.state[params[0]]['step']) == 4.0
    assert 'scales' in opt.state[params[2]] and 'scales' not in opt.state[params[0]]
    for p in params:
        p.grad = None
    before = snapshot(opt, params)
    opt.step()
    assert all(np.array_equal(a['p'], b['p']) for a, b in zip(snapshot(opt, params), before))


@pytest.mark.parametrize('bits', [32, 8])
def test_values_that_are_not_finite_stay_where_they_are(optim, bits):
    """Without a clip one element's infinity or NaN is that element's alone; an 8-bit block keeps the others' codes."""
    clean, dirty = make([3000], torch.float32), make([3000], torch.float32)
    dirty[0].grad[5], dirty[0].grad[300], dirty[0].grad[301] = float('nan'), float('inf'), -float('inf')
    opts = [optim.AdamW(p, **HYPER, state_bits=bits, min_8bit_numel=1) for p in (clean, dirty)]
    for p in (clean, dirty):
        p[0].grad[7] = 0.0
    for _ in range(2):
        for o in opts:
            o.step()
    bad = torch.zeros(3000, dtype=torch.bool)
    bad[[5, 300, 301]] = True
    (sa, sb), k2 = (o.state[p[0]] for o, p in zip(opts, (clean, dirty))), 'exp_avg_sq' if bits == 32 else 'exp_avg_root'
    for x, y in [(clean[0], dirty[0])] + [(sa[k], sb[k]) for k in ('exp_avg', k2)]:
        x, y = x.detach().float().cpu(), y.detach().float().cpu()
        if x.shape == (3000,):
            assert not torch.isfinite(y[bad]).any()
        keep = ~bad
        if bits == 8:                                # the bad elements may have held a block's largest value
            keep[:512] = False
            assert torch.isfinite(y[:512][~bad[:512]]).all()
        assert torch.equal(x[keep], y[keep])


def test_a_norm_that_is_not_finite_spreads_as_torchs_does(optim):
    for bad in (float('nan'), float('inf')):
        p = make([40, 600], torch.float32)
        p[0].grad[3] = bad
        q = [torch.nn.Parameter(x.detach().clone()) for x in p]
        for x, y in zip(p, q):
            y.grad = x.grad.clone()
        want = torch.nn.utils.clip_grad_norm_(q, 1.0)
        got = optim.clip_grad_norm_(p, 1.0)
        assert torch.equal(torch.isnan(want), torch.isnan(got)) and torch.equal(torch.isinf(want), torch.isinf(got))
        for x, y in zip(p, q):
            assert torch.equal(torch.isnan(x.grad), torch.isnan(y.grad))
        p[0].grad[3] = bad
        with pytest.raises(RuntimeError, match='not finite'):
            optim.clip_grad_norm_(p, 1.0, error_if_nonfinite=True)


def test_8bit_rounding_does_not_freeze_the_second_moment(optim):
    """With no gradient the root decays by sqrt(b2) a step; rounding to nearest would leave it where it is.  A step moves r by
    0.5 % where codes lie r / 16 apart at least, so it changes a code with probability p <= 0.08 and adds a variance of at most
    0.074 ulp^2, ulp <= 0.1 / 8: over 100 steps and 65536 elements the mean deviates by 1.3e-4, 0.22 % of it."""
    n, steps, b2 = 65536, 100, 0.99
    p = torch.nn.Parameter(torch.zeros(n, device='cuda'))
    p.grad = torch.full_like(p, 1.0)
    opt = optim.AdamW([p], lr=0.0, betas=(0.9, b2), state_bits=8)
    opt.step()
    p.grad = torch.zeros_like(p)
    for _ in range(steps):
        opt.step()
    st = opt.state[p]
    root = optim.dequantize_moment(st['exp_avg_root'], st['scales'][:, 1])
    want = math.sqrt((1 - b2) * b2 ** steps)
    assert abs(float(root.mean()) / want - 1) < 0.015
    assert float(root.min()) > 0


@pytest.mark.parametrize('bits', [32, 8])
def test_gradients_of_any_magnitude(optim, bits):
    """Blocks of 1e-30 (squares vanish) to 1e17 (the largest whose square fp32 holds in v), zeros among them."""
    mags = [1e-30, 1e-24, 1e-22, 3e-20, 1e-18, 1e-12, 1.0, 1e9, 1e17]
    g = torch.Generator().manual_seed(11)
    p = torch.nn.Parameter(torch.randn(256 * len(mags), generator=g).cuda())
    opt = optim.AdamW([p], **HYPER, state_bits=bits, min_8bit_numel=1)
    for _ in range(3):
        grad = torch.randn(len(mags), 256, generator=g) * torch.tensor(mags, dtype=torch.float64)[:, None]
        grad[:, ::5] = 0.0
        p.grad = grad.float().view(-1).cuda()
        before = snapshot(opt, [p])
        opt.step()
        check_step([p], before, snapshot(opt, [p]), HYPER)


# ------------------------------------------------------------------------------------------ layouts, streams, graphs
@pytest.mark.parametrize('bits', [32, 8])
def test_channels_last_parameters_and_a_change_of_layout(optim, bits):
    g = torch.Generator().manual_seed(4)
    w = torch.randn(24, 40, 3, 3, generator=g)
    grads = [torch.randn(24, 40, 3, 3, generator=g) for _ in range(3)]
    a = torch.nn.Parameter(w.cuda())
    b = torch.nn.Parameter(w.cuda().to(memory_format=torch.channels_last))
    oa, ob = (optim.AdamW([p], **HYPER, state_bits=bits, min_8bit_numel=1) for p in (a, b))
    for k, gr in enumerate(grads):
        a.grad = gr.cuda()
        b.grad = gr.cuda() if k != 1 else gr.cuda().to(memory_format=torch.channels_last)     # like its parameter, or not
        if k == 2:                                                                            # net.to(memory_format=...) later
            a.data = a.data.to(memory_format=torch.channels_last)
            b.data = b.data.contiguous()
        before = snapshot(ob, [b])
        if k < 2:
            before[0]['g'] = mem(torch.empty_like(b).copy_(b.grad))
            oa.step(), ob.step()
            check_step([b], before, snapshot(ob, [b]), HYPER)
        else:
            oa.step(), ob.step()
    assert ob.state[b]['exp_avg'].stride() == b.stride()
    if bits == 32:
        assert torch.equal(a, b) and torch.equal(oa.state[a]['exp_avg'], ob.state[b]['exp_avg'])
    else:
        # the third step starts from moments that were rounded to nearest in another order's blocks: 2^-4 of each, and a
        # sixteenth of m and of the root moves a step of at most lr * 2.4 (three steps, b2 = 0.99) by less than an eighth, twice
        assert float((a.detach() - b.detach()).abs().max()) <= 3 * 2 * HYPER['lr'] * 2.4


def test_another_stream(optim):
    params, twin = make([200001, 50], torch.float32), make([200001, 50], torch.float32)
    opt, ref = (optim.AdamW(p, **HYPER, max_norm=0.1, state_bits=8) for p in (params, twin))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(5):
            opt.step()
            optim.clip_grad_norm_(params, 1e9)
    torch.cuda.current_stream().wait_stream(s)
    for _ in range(5):
        ref.step()
    assert all(torch.equal(a, b) for a, b in zip(params, twin)) and torch.equal(opt.total_norm, ref.total_norm)


@pytest.mark.parametrize('bits', [32, 8])
def test_a_captured_step_counts_and_follows_the_learning_rate(optim, bits):
    sizes = [70001, 300, 5]
    params, twin = make(sizes, torch.float32), make(sizes, torch.float32)
    lr = torch.tensor(1e-2, device='cuda')
    kw = dict(HYPER, max_norm=0.2, state_bits=bits, seed=5)
    opt, ref = optim.AdamW(params, **dict(kw, lr=lr)), optim.AdamW(twin, **kw)
    with pytest.raises(RuntimeError, match='before capturing'):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            opt.step()
    opt.step(), ref.step()
    graph, scratch = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    norm = opt.total_norm
    if bits == 32:                                                    # what a replay would do over and over is refused
        w = torch.nn.Parameter(torch.randn(8, 8, 3, 3, device='cuda'))
        w.grad = torch.randn_like(w)
        other = optim.AdamW([w])
        other.step()
        w.data = w.data.to(memory_format=torch.channels_last)
        with pytest.raises(RuntimeError, match='before capturing'):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                other.step()
    with torch.cuda.graph(scratch):                                   # another graph's scratch is its own
        optim.clip_grad_norm_(twin, 1e9)
    for k in range(4):
        rate = 1e-2 / (k + 1)
        lr.fill_(rate)
        ref.param_groups[0]['lr'] = float(lr)
        for p, q in zip(params, twin):
            new = torch.randn_like(p) * 10.0 ** -k
            p.grad.copy_(new), q.grad.copy_(new)
        graph.replay()
        ref.step()
        scratch.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(params, twin)), k
        assert torch.equal(norm, ref.total_norm)
        assert float(opt.state[params[0]]['step']) == float(ref.state[twin[0]]['step']) == k + 2
    for p, q in zip(params, twin):
        for key, x in opt.state[p].items():
            y = ref.state[q][key]
            assert torch.equal(x.view(torch.uint8), y.view(torch.uint8)) if x.element_size() == 1 else torch.equal(x, y)


def test_grad_scaler_skips_on_the_device(optim):
    params, twin = make([5000, 40], torch.float32), make([5000, 40], torch.float32)
    opt, ref = optim.AdamW(params, **HYPER, max_norm=0.1), optim.AdamW(twin, **HYPER, max_norm=0.1)
    scaler = torch.amp.GradScaler('cuda', init_scale=1024.0)
    scaler.scale(torch.zeros((), device='cuda'))
    for k, (overflow, unscale) in enumerate([(False, False), (True, False), (False, True), (True, True), (False, False)]):
        for p, q in zip(params, twin):
            new = torch.randn_like(p)
            p.grad, q.grad = new * float(scaler.get_scale()), new.clone()
        if overflow:
            params[1].grad[3] = float('inf')
        if unscale:
            scaler.unscale_(opt)
        kept = [p.detach().clone() for p in params]
        scaler.step(opt)
        scaler.update()
        if overflow:
            assert all(torch.equal(p, q) for p, q in zip(params, kept))
        else:
            ref.step()
            assert all(torch.equal(p, q) for p, q in zip(params, twin)), k      # the scales are powers of two
    assert float(opt.state[params[0]]['step']) == 3.0
    assert not hasattr(opt, 'found_inf')


def test_two_optimizers_take_turns(optim):
    """Scratch belongs to a call: interleaved steps of two optimizers give what each gives alone."""
    def one():
        p = make([30001, 77], torch.float32, seed=8)
        return p, optim.AdamW(p, **HYPER, max_norm=0.3, state_bits=8)
    a, b, c = one(), one(), one()
    for _ in range(3):
        a[1].step(), b[1].step()
    for _ in range(3):
        c[1].step()
    for x in (a, b):
        assert all(torch.equal(p, q) for p, q in zip(x[0], c[0]))


# ---------------------------------------------------------------------------------------------------- checkpoints
def test_32bit_checkpoints_are_torchs(optim):
    a, b, c = (make([300, 4097], torch.float32) for _ in range(3))
    kw = dict(HYPER)
    ours, stock, third = optim.AdamW(a, **kw), torch.optim.AdamW(b, **kw), optim.AdamW(c, **dict(kw, lr=5.0))
    for _ in range(2):
        ours.step(), stock.step()
    for p, q in zip(a, b):
        assert torch.allclose(p, q, rtol=1e-5, atol=1e-7)
    sd = ours.state_dict()
    assert set(sd['state'][0]) == {'step', 'exp_avg', 'exp_avg_sq'}
    b2 = [torch.nn.Parameter(p.detach().clone()) for p in a]
    stock2 = torch.optim.AdamW(b2, **kw)
    stock2.load_state_dict(copy.deepcopy({**sd, 'param_groups': [{**stock2.state_dict()['param_groups'][0]}]}))
    for p, q in zip(c, a):
        p.data.copy_(q.data)
    third.load_state_dict(stock2.state_dict())
    assert third.param_groups[0]['lr'] == kw['lr'] and third.state[c[0]]['step'].is_cuda
    for p, q, r in zip(b2, a, c):
        p.grad = q.grad = r.grad = torch.randn_like(q)
    ours.step(), stock2.step(), third.step()
    for p, q, r in zip(a, b2, c):
        assert torch.allclose(p, q, rtol=1e-5, atol=1e-7) and torch.equal(p, r)
    bad = copy.deepcopy(sd)
    bad['state'][0]['exp_avg'] = torch.zeros(299)
    with pytest.raises(ValueError, match='shape'):
        third.load_state_dict(bad)
    bad = copy.deepcopy(sd)
    bad['param_groups'][0]['amsgrad'] = True
    with pytest.raises(ValueError, match='amsgrad'):
        third.load_state_dict(bad)
    other = torch.optim.RMSprop(b2)
    other.step()
    with pytest.raises(ValueError, match='not the state'):
        third.load_state_dict(other.state_dict())
    with pytest.raises(ValueError, match='groups'):
        optim.AdamW(c[:1], **kw).load_state_dict(sd)
    lr = torch.tensor(7.0, device='cuda')                 # the tensor that a graph reads stays that tensor
    fourth = optim.AdamW(c, lr=lr)
    fourth.load_state_dict(sd)
    assert fourth.param_groups[0]['lr'] is lr and abs(float(lr) - kw['lr']) < 1e-9


def test_8bit_checkpoints_resume_to_the_bit_and_convert(optim, tmp_path):
    a, b = make([300, 70001], torch.bfloat16), make([300, 70001], torch.bfloat16)
    oa, ob = (optim.AdamW(p, **HYPER, state_bits=8, seed=3) for p in (a, b))
    for _ in range(3):
        oa.step()
    torch.save(oa.state_dict(), tmp_path / 'opt.pth')
    sd = torch.load(tmp_path / 'opt.pth', weights_only=True)
    for p, q in zip(b, a):
        p.data.copy_(q.data)
    ob.load_state_dict(sd)
    # into 32 bits: exactly what the codes stand for
    c = [torch.nn.Parameter(p.detach().clone()) for p in a]
    oc = optim.AdamW(c, **HYPER)
    oc.load_state_dict(sd)
    st = oa.state[a[1]]
    assert torch.equal(oc.state[c[1]]['exp_avg'], optim.dequantize_moment(st['exp_avg'], st['scales'][:, 0]))
    assert torch.equal(oc.state[c[1]]['exp_avg_sq'], optim.dequantize_moment(st['exp_avg_root'], st['scales'][:, 1]) ** 2)
    # and from 32 bits into 8: half a step of e4m3 (2^-4, 2^-10 of the scale among its subnormals)
    od = optim.AdamW([torch.nn.Parameter(p.detach().clone()) for p in a], **HYPER, state_bits=8)
    od.load_state_dict(oc.state_dict())
    sd2 = od.state[od.param_groups[0]['params'][1]]
    for k, col, ref in (('exp_avg', 0, oc.state[c[1]]['exp_avg']), ('exp_avg_root', 1, oc.state[c[1]]['exp_avg_sq'].sqrt())):
        unit = optim.dequantize_moment(torch.ones(70001, device='cuda').to(torch.float8_e4m3fn), sd2['scales'][:, col])
        assert ((optim.dequantize_moment(sd2[k], sd2['scales'][:, col]) - ref).abs() <= ref.abs() * 2.0 ** -4 + unit * 2.0 ** -9).all()
    oa.step(), ob.step()
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    for k in ('exp_avg', 'exp_avg_root', 'scales'):
        assert torch.equal(oa.state[a[1]][k].view(torch.uint8), ob.state[b[1]][k].view(torch.uint8))


def test_a_loaded_group_keeps_what_its_scheduler_put_there(optim):
    """Resuming a one-cycle run: the group's entries come back from either class's file, and the runs go on together."""
    sched = torch.optim.lr_scheduler.OneCycleLR

    def run(cls, params, steps, opt=None, file=None):
        opt = cls(params, lr=1e-3, betas=(0.9, 0.99))
        if file is not None:
            opt.load_state_dict(file['opt'])
        s = sched(opt, max_lr=1e-2, total_steps=20, last_epoch=-1 if file is None else 3)
        if file is not None:
            s.load_state_dict(file['sched'])
        rates = []
        for k in range(steps):
            for p in params:
                p.grad = torch.full_like(p, 0.1 + k)
            opt.step(), s.step()
            rates.append((opt.param_groups[0]['lr'], opt.param_groups[0]['betas'][0]))
        return rates, dict(opt=copy.deepcopy(opt.state_dict()), sched=s.state_dict()), opt

    want, _, _ = run(torch.optim.AdamW, make([300], torch.float32), 9)
    for first in (optim.AdamW, torch.optim.AdamW):
        for second in (optim.AdamW, torch.optim.AdamW):
            a, file, _ = run(first, make([300], torch.float32), 4)
            b, _, opt = run(second, make([300], torch.float32), 5, file=file)
            assert np.allclose(a + b, want, rtol=1e-12)
            assert opt.param_groups[0]['max_lr'] == 1e-2 and opt.param_groups[0]['initial_lr'] == file['opt']['param_groups'][0]['initial_lr']
    # what the file lacks stays (torch's knows no max_norm); what it holds is a copy and has to be sound
    opt = optim.AdamW(make([300], torch.float32), max_norm=0.5)
    _, file, _ = run(torch.optim.AdamW, make([300], torch.float32), 1)
    file['opt']['param_groups'][0]['notes'] = [1]
    opt.load_state_dict(file['opt'])
    file['opt']['param_groups'][0]['notes'].append(2)
    assert opt.param_groups[0]['max_norm'] == 0.5 and opt.param_groups[0]['notes'] == [1]
    for key, value in (('betas', (1.0, 0.9)), ('eps', -1.0), ('max_norm', 0.0)):
        bad = copy.deepcopy(file['opt'])
        bad['param_groups'][0].update({key: value, 'lr': 7.0})
        with pytest.raises(ValueError, match=key):
            opt.load_state_dict(bad)
        assert opt.param_groups[0]['lr'] != 7.0


@pytest.mark.parametrize('ours', [True, False])
def test_load_state_dict_calls_its_hooks(optim, ours):
    """As torch.optim.AdamW does: pre-hooks in turn, each on what the one before returned, then the load, then the others."""
    cls, seen = (optim if ours else torch.optim).AdamW, []
    opt = cls(make([300], torch.float32), lr=1e-3)
    opt.step()
    file = opt.state_dict()

    def change(o, sd):
        seen.append(('change', sd['param_groups'][0]['lr']))
        return {**sd, 'param_groups': [{**sd['param_groups'][0], 'lr': 0.5}]}

    def look(o, sd):
        seen.append(('look', sd['param_groups'][0]['lr']))
        sd['note'] = 1

    opt.register_load_state_dict_pre_hook(change)
    opt.register_load_state_dict_pre_hook(look)
    gone = opt.register_load_state_dict_pre_hook(lambda o, sd: seen.append('gone'))
    first = opt.register_load_state_dict_pre_hook(look, prepend=True)
    opt.register_load_state_dict_post_hook(lambda o: seen.append(('post', o.param_groups[0]['lr'])))
    gone.remove()
    opt.load_state_dict(file)
    assert seen == [('look', 1e-3), ('change', 1e-3), ('look', 0.5), ('post', 0.5)]
    assert file['param_groups'][0]['lr'] == 1e-3 and 'note' not in file and opt.param_groups[0]['lr'] == 0.5
    first.remove()
    copy.deepcopy(opt).load_state_dict(file)


@pytest.mark.parametrize('bits', [32, 8])
def test_a_file_whose_moments_do_not_fit_is_refused(optim, bits):
    """Neither spread over the parameter nor read as something else: every moment has the parameter's shape, codes are codes."""
    opt = optim.AdamW(make([300, 5000], torch.float32), state_bits=bits)
    opt.step()
    file = opt.state_dict()
    one = torch.ones(1, device='cuda')
    changes = [('exp_avg_sq', one), ('exp_avg_sq', torch.zeros((), device='cuda')), ('exp_avg', one)] if bits == 32 else [
        ('exp_avg', one.to(torch.float8_e4m3fn)), ('exp_avg_root', one.to(torch.float8_e4m3fn)), ('exp_avg_root', None),
        ('exp_avg', torch.zeros(5000, device='cuda')), ('exp_avg_root', torch.zeros(5000, dtype=torch.uint8, device='cuda')),
        ('scales', file['state'][1]['scales'][:1]), ('scales', file['state'][1]['scales'].view(torch.uint8)),
        ('scales', file['state'][1]['scales'][:, :1])]
    for target in (32, 8):
        other = optim.AdamW(make([300, 5000], torch.float32, 1), state_bits=target)
        other.step()
        params = other.param_groups[0]['params']
        before = snapshot(other, params)
        for key, value in changes:
            bad = copy.deepcopy(file)
            bad['state'][1][key] = value
            if value is None:
                del bad['state'][1][key]
            with pytest.raises(ValueError, match='load_state_dict'):
                other.load_state_dict(bad)
        for x, y in zip(before, snapshot(other, params)):
            assert x['t'] == y['t'] and np.array_equal(x['m'], y['m']) and np.array_equal(x['v'], y['v'])
        other.load_state_dict(file)


def test_copies_of_the_optimizer_and_a_state_that_leaves_the_device(optim):
    a = make([300, 70001], torch.float32)
    oa = optim.AdamW(a, **HYPER, state_bits=8, seed=3, max_norm=0.5)
    oa.step()
    b, ob = copy.deepcopy((a, oa))
    for p, q in zip(a, b):
        q.grad = p.grad
    c, oc = copy.deepcopy((a, oa))
    for p, q in zip(a, c):
        q.grad = p.grad
    oc.step()
    for st in oc.state.values():                          # offloaded between steps: the memory is really free, the step refused
        for k in list(st):
            st[k] = st[k].cpu()
    freed = torch.cuda.memory_allocated()
    with pytest.raises(RuntimeError, match='state'):
        oc.step()
    assert torch.cuda.memory_allocated() == freed
    for st in oc.state.values():
        for k in list(st):
            st[k] = st[k].cuda()
    oa.step(), ob.step(), oa.step(), ob.step(), oc.step()
    for p, q, r in zip(a, b, c):
        assert torch.equal(p, q) and torch.equal(p, r)


@pytest.mark.parametrize('bits', [32, 8])
def test_a_state_that_is_dropped_or_replaced_frees_its_memory(optim, bits):
    """The step's own bookkeeping holds neither the tensors nor the dictionaries they are in."""
    n = 1 << 22
    opt = optim.AdamW(make([n, 300], torch.float32), state_bits=bits)
    p = opt.param_groups[0]['params'][0]

    def freed(change):
        opt.step(), opt.step()
        held = torch.cuda.memory_allocated()
        change()
        return held - torch.cuda.memory_allocated()

    def off():
        opt.state[p] = {k: v.cpu() for k, v in opt.state[p].items()}

    at_least = n * 8 if bits == 32 else n * 2
    assert freed(off) >= at_least
    with pytest.raises(RuntimeError, match='state'):
        opt.step()
    opt.state[p] = {k: v.cuda() for k, v in opt.state[p].items()}
    assert freed(lambda: opt.state.pop(p)) >= at_least
    assert freed(opt.state.clear) >= at_least
    opt.step()
    assert float(opt.state[p]['step']) == 1.0
    # two parameters that exchange their states: each goes on with the other's moments, as the dictionary says
    a, b = make([400, 400], torch.float32)
    opt = optim.AdamW([a, b], **HYPER, state_bits=bits, min_8bit_numel=1)
    opt.step(), opt.step()
    opt.state[a], opt.state[b] = opt.state[b], opt.state[a]
    before = snapshot(opt, [a, b])
    opt.step()
    check_step([a, b], before, snapshot(opt, [a, b]), HYPER)


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason='one GPU')
def test_parameters_on_another_device_than_the_current_one(optim):
    p = make([5000, 40], torch.float32)
    q = [torch.nn.Parameter(x.detach().to('cuda:1')) for x in p]
    for x, y in zip(p, q):
        y.grad = x.grad.to('cuda:1')
    op, oq = optim.AdamW(p, **HYPER, max_norm=0.1, state_bits=8), optim.AdamW(q, **HYPER, max_norm=0.1, state_bits=8)
    for _ in range(2):
        op.step(), oq.step()
    assert float(optim.clip_grad_norm_(p, 0.01)) == float(optim.clip_grad_norm_(q, 0.01))
    for x, y in zip(p, q):
        assert torch.equal(x.cpu(), y.cpu()) and torch.equal(x.grad.cpu(), y.grad.cpu())


# --------------------------------------------------------------------------------------------------------- refusals
def test_refusals(optim):
    p = make([10, 20], torch.float32)
    with pytest.raises(ValueError, match='twice'):
        optim.AdamW([{'params': [p[0], p[0]]}])
    for kw in (dict(betas=(1.0, 0.9)), dict(betas=(0.9, -0.1)), dict(max_norm=0.0), dict(max_norm=-1.0)):
        with pytest.raises(ValueError):
            optim.AdamW(p, **kw)
    with pytest.raises(ValueError, match='same in each'):
        optim.AdamW([{'params': [p[0]], 'max_norm': 1.0}, {'params': [p[1]], 'max_norm': 2.0}])
    with pytest.raises(RuntimeError, match='float64'):
        optim.AdamW([torch.nn.Parameter(torch.zeros(3, dtype=torch.float64, device='cuda'))])
    with pytest.raises(RuntimeError, match='dense'):
        optim.AdamW([torch.nn.Parameter(torch.zeros(8, 8, device='cuda')[:, ::2])])
    opt = optim.AdamW(p)
    with pytest.raises(ValueError):
        opt.add_param_group({'params': [torch.nn.Parameter(torch.zeros(1, device='cuda'))], 'betas': (2.0, 0.1)})
    assert len(opt.param_groups) == 1
    opt.step()
    for key, value in (('step', torch.zeros(())), ('exp_avg', torch.zeros(10, device='cuda', dtype=torch.bfloat16)),
                       ('exp_avg_sq', torch.zeros(9, device='cuda'))):
        old, opt.state[p[0]][key] = opt.state[p[0]][key], value
        with pytest.raises(RuntimeError, match=key):
            opt.step()
        opt.state[p[0]][key] = old
    e = torch.nn.Parameter(torch.zeros(4, device='cuda'))
    e.grad = torch.zeros(1, device='cuda').expand(4)
    with pytest.raises(RuntimeError, match='dense'):
        optim.clip_grad_norm_([e], 1.0)
    with pytest.raises(ValueError, match='twice'):
        optim.clip_grad_norm_([p[0], p[0]], 1.0)
    opt.param_groups[0]['lr'] = torch.tensor(1e-3, dtype=torch.float64, device='cuda')
    with pytest.raises(RuntimeError, match='lr'):
        opt.step()


@pytest.mark.parametrize('key,value,error', [
    ('lr', torch.tensor(1e-3, dtype=torch.float64), None), ('lr', 'fast', ValueError), ('betas', (0.9,), ValueError),
    ('betas', (0.9, None), TypeError), ('eps', None, TypeError), ('weight_decay', 'none', ValueError), ('max_norm', -1.0, ValueError),
    ('max_norm', float('nan'), ValueError), ('max_norm', 0.0, ValueError)])
def test_a_step_that_fails_has_not_counted(optim, key, value, error):
    """What is wrong with the last group is found before the first group's launch."""
    a, b = make([5000, 3], torch.float32), make([40], torch.float32, 1)
    opt = optim.AdamW([{'params': a}, {'params': b}], **HYPER, max_norm=0.5)
    opt.step()
    good = opt.param_groups[1][key]
    before = snapshot(opt, a + b)
    for g in opt.param_groups[0 if key == 'max_norm' else 1:]:
        g[key] = value.cuda() if torch.is_tensor(value) else value
    with pytest.raises(error or RuntimeError):
        opt.step()
    after = snapshot(opt, a + b)
    for x, y in zip(before, after):
        assert x['t'] == y['t'] == 1.0 and all(np.array_equal(x[k], y[k]) for k in 'pmv')
    for g in opt.param_groups:
        g[key] = good
    opt.step()
    check_step(a + b, before, snapshot(opt, a + b), HYPER, 0.5, 0, opt.total_norm)


def test_a_limit_of_one_group_alone_is_refused_at_the_step(optim):
    a, b = make([5000, 3], torch.float32), make([40], torch.float32, 1)
    opt = optim.AdamW([{'params': a}, {'params': b}], **HYPER)
    for first, second in ((None, 0.5), (0.5, None), (0.5, 0.25)):
        opt.param_groups[0]['max_norm'], opt.param_groups[1]['max_norm'] = first, second
        before = snapshot(opt, a + b)
        with pytest.raises(ValueError, match='same in each'):
            opt.step()
        assert all(x['t'] == y['t'] and np.array_equal(x['p'], y['p']) for x, y in zip(before, snapshot(opt, a + b)))
    for g in opt.param_groups:                                        # in both it is the clip, as from the start
        g['max_norm'] = 0.25
    before = snapshot(opt, a + b)
    opt.step()
    check_step(a + b, before, snapshot(opt, a + b), HYPER, 0.25, 0, opt.total_norm)


@pytest.mark.parametrize('bits', [32, 8])
def test_tensors_that_share_memory_are_refused(optim, bits):
    """Two workgroups would write the same elements in any order."""
    def fresh():
        params = make([5000, 5000, 300], torch.float32)
        opt = optim.AdamW(params, **HYPER, state_bits=bits)
        opt.step()
        return params, opt

    def tied(ps, o):
        ps[1].data = ps[0].data

    def partly(ps, o):
        buf = torch.zeros(9999, device='cuda')
        ps[0].data, ps[1].data = buf[:5000], buf[4999:]

    def one_count(ps, o):
        o.state[ps[0]]['step'] = o.state[ps[2]]['step']

    def one_moment(ps, o):
        o.state[ps[0]]['exp_avg'] = o.state[ps[1]]['exp_avg']

    def own_moments(ps, o):
        o.state[ps[2]]['exp_avg_sq'] = o.state[ps[2]]['exp_avg']

    def parameter_as_moment(ps, o):
        o.state[ps[2]]['exp_avg'] = ps[2].data

    changes = [tied, partly, one_count, one_moment, own_moments, parameter_as_moment]
    if bits == 8:
        def one_scale(ps, o):
            o.state[ps[0]]['scales'] = o.state[ps[1]]['scales']
        changes.append(one_scale)
    for change in changes:
        params, opt = fresh()
        change(params, opt)
        before = snapshot(opt, params)
        for _ in range(2):
            with pytest.raises(RuntimeError, match='overlap'):
                opt.step()
        for x, y in zip(before, snapshot(opt, params)):
            assert x['t'] == y['t'] == 1.0 and all(np.array_equal(x[k], y[k]) for k in 'pmv')
    # side by side is apart
    params, opt = fresh()
    buf = torch.randn(10000, device='cuda')
    params[0].data, params[1].data = buf[:5000], buf[5000:]
    before = snapshot(opt, params)
    opt.step()
    check_step(params, before, snapshot(opt, params), HYPER)


@pytest.mark.parametrize('bits', [32, 8])
def test_the_smallest_eps(optim, bits):
    """Elements whose gradient is always zero stay (but for the decay) whatever eps is above zero; below fp32's normal numbers it is
    refused with 8 bits, before anything has counted."""
    for eps in (2.0 ** -126, 1e-30) + ((1e-40,) if bits == 32 else ()):
        hyper = dict(HYPER, eps=eps)
        params = make([5000], torch.float32)
        params[0].grad[::3] = 0.0
        opt = optim.AdamW(params, **hyper, state_bits=bits, min_8bit_numel=1)
        for _ in range(2):
            before = snapshot(opt, params)
            opt.step()
            check_step(params, before, snapshot(opt, params), hyper)
    if bits == 8:
        with pytest.raises(ValueError, match='eps'):
            optim.AdamW(params, eps=1e-40, state_bits=8)
        opt.param_groups[0]['eps'] = 1e-40
        with pytest.raises(ValueError, match='eps'):
            opt.step()
        assert float(opt.state[params[0]]['step']) == 2.0
        opt.param_groups[0]['eps'] = 1e-8
        opt.step()


# ------------------------------------------------------------------------------------------------------------- clip
@pytest.mark.parametrize('sizes', list(SIZES))
@pytest.mark.parametrize('dtype', list(TYPES) + ['mixed'])
def test_clip_grad_norm(optim, sizes, dtype):
    if dtype == 'mixed':
        params = [q for i, n in enumerate(SIZES[sizes]) for q in make([n], list(TYPES.values())[i % 3], seed=i)]
    else:
        params = make(SIZES[sizes], TYPES[dtype])
    before = [mem(p.grad) for p in params]
    norm = O.norm(before)
    for limit in (norm * 0.37, norm * 2, math.inf, 0.0):
        for p, b in zip(params, before):
            p.grad.copy_(torch.from_numpy(b).to(p.dtype))
        got = optim.clip_grad_norm_(params, limit)
        assert got.dtype == torch.float32 and got.is_cuda and abs(float(got) - norm) <= 3 * O.U * norm
        c = O.clip_coef(norm, limit)
        for p, b in zip(params, before):
            fi = torch.finfo(p.dtype)
            err = np.abs(b * c) * (COEF_ERR + O.U + fi.eps / 2) + fi.eps / 2 * fi.smallest_normal
            assert (np.abs(mem(p.grad) - b * c) <= (err if c < 1 else 0)).all()


def test_clip_of_huge_and_tiny_gradients(optim):
    """Squares beyond fp32's range: the norm is still the norm."""
    for value in (1e30, 1e-30):
        p = torch.nn.Parameter(torch.zeros(1000, device='cuda'))
        p.grad = torch.full_like(p, value)
        got = float(optim.clip_grad_norm_([p], value))
        want = float(np.float32(value)) * math.sqrt(1000)
        assert abs(got - want) <= 3 * O.U * want


def test_a_norm_beyond_fp32_is_not_finite(optim):
    """A thousand times 1e38: the sum of squares is finite in fp64, the fp32 norm that divides the gradients is not."""
    for dtype in (torch.float32, torch.bfloat16):
        p = [torch.nn.Parameter(torch.zeros(n, dtype=dtype, device='cuda')) for n in (1000, 7)]
        for q in p:
            q.grad = torch.full_like(q, 1e38)
        kept = [q.grad.clone() for q in p]
        with pytest.raises(RuntimeError, match='not finite'):
            optim.clip_grad_norm_(p, 1.0, error_if_nonfinite=True)
        assert all(torch.equal(q.grad, k) for q, k in zip(p, kept))
        for q in p:
            q.grad.fill_(1e37)
        got = float(optim.clip_grad_norm_(p, 1.0, error_if_nonfinite=True))
        want = float(p[0].detach().new_tensor(1e37)) * math.sqrt(1007)
        assert abs(got - want) <= 3 * O.U * want


def test_gradients_that_share_memory_are_not_clipped(optim):
    """They would be scaled once or twice, as the workgroups come; side by side in any order they are apart."""
    params = [torch.nn.Parameter(torch.zeros(n, device='cuda')) for n in (5000, 5000, 300, 0)]
    for starts in ((0, 0, 9000, 0), (0, 4999, 12000, 9), (9000, 6000, 8700, 3), (9000, 3000, 8750, 0)):
        buf = torch.randn(20000, device='cuda')
        for p, a in zip(params, starts):
            p.grad = buf[a:a + p.numel()]
        kept = buf.clone()
        with pytest.raises(RuntimeError, match='overlap'):
            optim.clip_grad_norm_(params, 1.0)
        assert torch.equal(buf, kept)
    for starts in ((0, 5000, 10000, 7), (5300, 300, 0, 7), (300, 5300, 0, 7), (5000, 0, 10000, 7)):
        buf = torch.randn(20000, device='cuda')
        for p, a in zip(params, starts):
            p.grad = buf[a:a + p.numel()]
        kept = f64(buf)
        want = O.norm([kept[:10300]])
        got = optim.clip_grad_norm_(params, 1.0)
        assert abs(float(got) - want) <= 3 * O.U * want
        c = O.clip_coef(want, 1.0)
        assert (np.abs(f64(buf)[:10300] - kept[:10300] * c) <= np.abs(kept[:10300] * c) * (COEF_ERR + 2 * O.U)).all()
        assert np.array_equal(f64(buf)[10300:], kept[10300:])


def test_more_than_two_to_the_31_elements(optim):
    """Offsets beyond 32 bits: the last elements of a tensor of 2^31 + 4099."""
    n, tail = 2 ** 31 + 4099, 5000
    p = torch.nn.Parameter(torch.zeros(n, dtype=torch.bfloat16, device='cuda'))
    p.grad = torch.zeros(n, dtype=torch.bfloat16, device='cuda')
    g = torch.randn(tail, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16)
    p.grad[-tail:] = g.cuda()
    opt = optim.AdamW([p], **HYPER, state_bits=8, max_norm=1.0, seed=9)
    opt.step()
    want_norm = O.norm([f64(g)])
    assert abs(float(opt.total_norm) - want_norm) <= 3 * O.U * want_norm
    c = O.clip_coef(want_norm, 1.0)
    fi = torch.finfo(torch.bfloat16)
    want = O.step(np.zeros(tail), f64(g), np.zeros(tail), np.zeros(tail), 1, HYPER['lr'], *HYPER['betas'], 1e-8, 0.1, c, COEF_ERR,
                  fi.eps / 2, fi.smallest_normal)
    assert (np.abs(f64(p[-tail:]) - want['p']) <= want['pe']).all()
    assert not p[:-tail].any()
    st = opt.state[p]
    first = (n - tail) // 256 * 256                                   # whole blocks from here
    lead = n - tail - first
    k = st['scales'].view(torch.uint8)[first // 256:].cpu().numpy().astype(int) - 127
    for key, col, x, xe, u in (('exp_avg', 0, want['m'], want['me'], O.fractions(n - first, 1, 9, first)[0]),
                               ('exp_avg_root', 1, want['r'], want['re'], O.fractions(n - first, 1, 9, first)[1])):
        x, xe = (np.concatenate([np.zeros(lead), y]) for y in (x, xe))
        xe[:lead] = 0
        lo, hi = O.code_range(x, xe, k[:, col], u, col == 1)
        codes = f64(st[key][first:].float())
        assert (lo <= codes).all() and (codes <= hi).all()


# ------------------------------------------------------------------------------------------------------- the trainer
def test_the_trainer_steps_with_it(optim):
    """Trainer(optimizer='adamw') on the flat gradient buffer against torch.optim.AdamW fed with the same gradients; 8 bits
    moves the same way; the checkpoint is numbered in net.parameters() order."""
    from test_gpu_trainstep import _closed_form, _img, SHAPE
    from unet import UNet
    from unetk.trainer import Trainer
    img = _img()
    mask = (torch.arange(SHAPE[0] * SHAPE[2] * SHAPE[3], device='cuda') % 7 == 0).long().view(SHAPE[0], SHAPE[2], SHAPE[3])
    net = _closed_form(UNet(3, 2, False)).cuda().to(memory_format=torch.channels_last).train()
    twin = [torch.nn.Parameter(p.detach().clone().contiguous()) for p in net.parameters()]
    tr = Trainer(net, amp=False, learning_rate=1e-4, weight_decay=0.01, optimizer='adamw')
    stock = torch.optim.AdamW(twin, lr=1e-4, weight_decay=0.01)
    for _ in range(2):
        tr.step(img, mask)
        for p, q in zip(net.parameters(), twin):
            q.grad = tr.sync.views[p].detach().clone()
        norm = torch.nn.utils.clip_grad_norm_(twin, 1.0)
        assert abs(float(norm) - float(tr.optimizer.total_norm)) <= 1e-5 * float(norm)
        stock.step()
        for p, q in zip(net.parameters(), twin):
            # the same gradients: the decay, the difference and the store round a parameter three times on each side and step, and
            # a step of at most lr / (1 - beta1) carries the moments' roundings, some 10 of 2^-24
            assert ((p - q).abs() <= 12 * 2.0 ** -24 * q.abs() + 2 * 20 * 2.0 ** -24 * 1e-3).all()
    sd = tr.optimizer.state_dict()
    for i, q in enumerate(twin):
        assert sd['state'][i]['exp_avg'].shape == q.shape
    for kw in (dict(optimizer='sgd'), dict(state_bits=8), dict(optimizer='adamw', state_bits=8, fused_optimizer=False)):
        with pytest.raises(ValueError, match='optimizer'):
            Trainer(net, **kw)
    # the same loop around a stock optimizer, with the clip by itself
    net2 = _closed_form(UNet(3, 2, False)).cuda().to(memory_format=torch.channels_last).train()
    tr2 = Trainer(net2, amp=False, learning_rate=1e-4, weight_decay=0.01, optimizer='adamw', fused_optimizer=False)
    tr2.step(img, mask)
    total = sum(float(p.grad.double().square().sum()) for p in net2.parameters()) ** 0.5
    assert total <= 1.0 + 1e-5 and type(tr2.optimizer) is torch.optim.AdamW


@pytest.mark.parametrize('amp_dtype', [torch.bfloat16, torch.float16])
def test_the_trainer_in_mixed_precision_with_8bit_moments(optim, amp_dtype):
    from test_gpu_trainstep import _closed_form, _img, SHAPE
    from unet import UNet
    from unetk.trainer import Trainer
    img = _img()
    mask = (torch.arange(SHAPE[0] * SHAPE[2] * SHAPE[3], device='cuda') % 7 == 0).long().view(SHAPE[0], SHAPE[2], SHAPE[3])
    net = _closed_form(UNet(3, 2, False)).cuda().to(memory_format=torch.channels_last).train()
    tr = Trainer(net, learning_rate=1e-4, weight_decay=0.01, optimizer='adamw', state_bits=8, amp_dtype=amp_dtype)
    for k in range(2):
        before = snapshot(tr.optimizer, list(net.parameters()))
        tr.step(img, mask)
        params = list(net.parameters())
        for b, p in zip(before, params):
            b['g'] = f64(tr.sync.views[p])
        check_step(params, before, snapshot(tr.optimizer, params), dict(lr=1e-4, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01),
                   1.0, 0, tr.optimizer.total_norm)
    kinds = {'scales' in tr.optimizer.state[p] for p in net.parameters()}
    assert kinds == {True, False}


# ------------------------------------------------------------------------------- what is carried from step to step
@pytest.mark.parametrize('bits', [32, 8])
def test_whatever_moves_between_steps_is_noticed(optim, bits):
    """The checks of one step serve the next; everything that may change in between has to end that.  The twin forgets them
    before each step."""
    sizes = [5000, 12, 4097, 300]
    params, twin = make(sizes, torch.float32), make(sizes, torch.float32)
    kw = dict(HYPER, max_norm=0.3, state_bits=bits)
    opt, ref = optim.AdamW(params, **kw), optim.AdamW(twin, **kw)
    g = torch.Generator().manual_seed(6)
    hold = []

    def new_data(o, ps):
        hold.append(ps[0].data)
        ps[0].data = ps[0].data.clone() * 0.5

    def new_entry(o, ps):
        hold.append(o.state[ps[2]]['exp_avg'])
        x = o.state[ps[2]]['exp_avg']
        o.state[ps[2]]['exp_avg'] = torch.zeros_like(x) if bits == 32 else torch.zeros_like(x, dtype=torch.uint8).view(x.dtype)

    def moved_entry(o, ps):
        o.state[ps[1]]['exp_avg_sq'].data = o.state[ps[1]]['exp_avg_sq'].data.clone()
        o.state[ps[1]]['exp_avg_sq'].mul_(2.0)

    def new_state(o, ps):
        o.state[ps[3]] = {k: v.clone() for k, v in o.state[ps[3]].items()}
        o.state[ps[3]]['step'].fill_(7.0)

    def no_state(o, ps):
        hold.append(o.state.pop(ps[1]))

    def no_gradient(o, ps):
        ps[2].grad = None

    def strided_gradient(o, ps):
        ps[0].grad = torch.stack([ps[0].grad, -ps[0].grad], 1)[:, 0]

    def new_group(o, ps):
        ps.append(make([4500], torch.float32, seed=12)[0])
        o.add_param_group({'params': [ps[-1]], 'lr': 0.5, 'betas': (0.5, 0.6)})

    def other_parameter(o, ps):
        hold.append(ps[1])
        ps[1] = make([12], torch.float32, seed=13)[0]
        o.param_groups[0]['params'][1] = ps[1]

    def a_note(o, ps):
        o.state[ps[0]]['note'] = 'kept by the user'

    def new_rate(o, ps):
        o.param_groups[0]['lr'] *= 3
        o.param_groups[0]['betas'] = (0.5, 0.9)

    for change in (None, new_data, None, new_entry, moved_entry, new_state, no_state, no_gradient, None, strided_gradient, new_group,
                   new_rate, other_parameter, a_note, None):
        for i in range(len(params)):
            new = torch.randn(params[i].numel(), generator=g).cuda()
            params[i].grad, twin[i].grad = new, new.clone()
        if change is not None:
            change(opt, params), change(ref, twin)
        ref._plan = None
        opt.step(), ref.step()
        assert all(torch.equal(p, q) for p, q in zip(params, twin)), change
        assert [float(opt.state[p]['step']) for p in params] == [float(ref.state[q]['step']) for q in twin], change
    assert float(opt.state[params[3]]['step']) == 17.0 and float(opt.state[params[2]]['step']) == 14.0
    for o, ps in ((opt, params), (ref, twin)):
        ps[0].data = ps[0].data.cpu()
        with pytest.raises(RuntimeError, match='cuda'):
            o.step()


def test_a_parameter_that_was_cut_is_refused_until_all_else_is(optim):
    params = make([5000, 300], torch.float32)
    opt = optim.AdamW(params, **HYPER)
    opt.step()
    whole = params[0].data
    params[0].data = whole[:4000]
    for _ in range(2):
        with pytest.raises(RuntimeError, match='shape'):
            opt.step()
    params[0].grad = params[0].grad[:4000].clone()
    with pytest.raises(RuntimeError, match='state'):
        opt.step()
    for k in ('exp_avg', 'exp_avg_sq'):
        opt.state[params[0]][k] = opt.state[params[0]][k][:4000]
    before, kept = snapshot(opt, params), whole[4000:].clone()
    opt.step()
    check_step(params, before, snapshot(opt, params), HYPER)
    assert torch.equal(whole[4000:], kept)


def test_frozen_parameters_of_a_flat_buffer_stay(optim):
    from unet import UNet
    from unetk.ddp import FlatGrads
    torch.manual_seed(0)
    net = UNet(3, 2, False).cuda()
    fg = FlatGrads(net, grads_to_autograd=False)
    opt = optim.AdamW(fg, lr=1e-2, weight_decay=0.5)
    with pytest.raises(RuntimeError, match='no gradients'):
        opt.step()
    with pytest.raises(ValueError, match='no place'):
        opt.add_param_group({'params': make([10], torch.float32)})
    frozen = net.inc.double_conv[0].weight
    for k in range(4):
        frozen.requires_grad_(k == 2)
        fg.initial_grads()
        fg.flat.normal_()
        before = frozen.detach().clone(), net.outc.conv.weight.detach().clone()
        opt.step()
        assert torch.equal(frozen, before[0]) == (k != 2) and not torch.equal(net.outc.conv.weight, before[1])
    assert float(opt.state[frozen]['step']) == 1.0 and float(opt.state[net.outc.conv.weight]['step']) == 4.0
