"""The optimizer-step operators as a training loop calls them, their plain forms and the work they cannot do without.

An AdamW step over all parameters of a network at once, its moments in 32 bits or in 8, with the global-norm clip in
front; and the clip by itself.  The parameter lists are those of the repository's U-Net at several widths, one part of
it (a head or a layer that is tuned alone), and lists of tensors of arbitrary sizes.
"""
import math
import os
import sys

import torch

own = False

BLOCK = 256                    # elements that share one scale per moment in the 8-bit form
MIN_8BIT = 4096                # smaller tensors keep 32-bit moments
TYPES = {'fp32': torch.float32, 'bf16': torch.bfloat16, 'fp16': torch.float16}
MASK = 0xFFFFFFFF


# ---------------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # only OutConv is tuned: 130 values in two tensors, a step is all launch latency
        dict(name='adamw32_head', op='adamw', bits=32, kind='head', width=64, dtype='fp32', max_norm=0.0, age=40,
             lr=1e-4, beta2=0.999),
        # the full network as the trainer steps it: 31 M fp32 parameters, clip to 1
        dict(name='adamw32_unet', op='adamw', bits=32, kind='unet', width=64, dtype='fp32', max_norm=1.0, age=2000,
             lr=1e-5, beta2=0.999),
        # the bilinear network held in bf16
        dict(name='adamw32_bilinear_bf16', op='adamw', bits=32, kind='bilinear', width=64, dtype='bf16', max_norm=1.0,
             age=300, lr=1e-4, beta2=0.99),
        # many tensors of any size, one behind the other without padding, each with an age of its own
        dict(name='adamw32_ragged', op='adamw', bits=32, kind='ragged', tensors=190, largest=300001, dtype='fp32',
             max_norm=0.0, age=700, lr=1e-4, beta2=0.999),
        # twice the width: 124 M parameters, the largest step
        dict(name='adamw32_wide', op='adamw', bits=32, kind='unet', width=128, dtype='fp32', max_norm=1.0, age=9000,
             lr=1e-5, beta2=0.999),
        # one convolution tuned alone with 8-bit moments
        dict(name='adamw8_layer', op='adamw', bits=8, kind='layer', width=64, dtype='fp32', max_norm=0.0, age=25,
             lr=1e-5, beta2=0.999),
        dict(name='adamw8_unet', op='adamw', bits=8, kind='unet', width=64, dtype='fp32', max_norm=1.0, age=2000,
             lr=1e-5, beta2=0.999),
        dict(name='adamw8_ragged_fp16', op='adamw', bits=8, kind='ragged', tensors=70, largest=1500007, dtype='fp16',
             max_norm=1.0, age=150, lr=1e-5, beta2=0.99),
        dict(name='adamw8_wide_bf16', op='adamw', bits=8, kind='unet', width=128, dtype='bf16', max_norm=1.0, age=9000,
             lr=1e-5, beta2=0.999),
        # gradient clipping in front of somebody else's optimizer
        dict(name='clip_layer', op='clip', kind='layer', width=64, dtype='fp32', max_norm=1.0),
        dict(name='clip_unet', op='clip', kind='unet', width=64, dtype='fp32', max_norm=1.0),
        dict(name='clip_ragged_bf16', op='clip', kind='ragged', tensors=130, largest=2500009, dtype='bf16', max_norm=1.0),
    ]


def draw(rng):
    def log_int(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    case = dict(op=rng.choice(['adamw', 'adamw', 'adamw', 'clip']), dtype=rng.choice(['fp32', 'fp32', 'bf16', 'fp16']),
                kind=rng.choice(['unet', 'bilinear', 'ragged', 'ragged', 'layer']))
    if case['kind'] == 'ragged':
        case['tensors'] = log_int(1, 200)
        case['largest'] = log_int(1, 6000000)
    else:
        case['width'] = log_int(5, 112)
    if case['op'] == 'adamw':
        case['bits'] = rng.choice([32, 8])
        case['age'] = log_int(1, 20000)
        case['lr'] = rng.choice([1e-5, 2e-5, 5e-6])
        case['beta2'] = rng.choice([0.999, 0.99, 0.95])
    case['max_norm'] = rng.choice([0.0, 1.0, 0.25]) if case['op'] == 'adamw' else rng.choice([1.0, 0.25])
    return case


def sizes(case):
    """Elements of each tensor of the case's list."""
    kind = case['kind']
    if kind == 'ragged':                                  # sizes spread over their logarithm, in a fixed shuffled order
        t, top = case['tensors'], math.log(case['largest'])
        return [max(1, int(math.exp(top * (1.0 if i == 0 else ((i * 0.6180339887) % 1.0) ** 0.7)))) for i in range(t)]
    b = case['width']
    if kind == 'head':
        return [2 * b, 2]
    if kind == 'layer':
        return [b * b * 9]
    f = 2 if kind == 'bilinear' else 1

    def double(ci, mid, co):
        return [mid * ci * 9, mid, mid, co * mid * 9, co, co]

    out = double(3, b, b)
    for k, c in enumerate((b, 2 * b, 4 * b, 8 * b)):
        co = 2 * c // (f if k == 3 else 1)
        out += double(c, co, co)
    for k, c in enumerate((16 * b, 8 * b, 4 * b, 2 * b)):
        if f == 1:
            out += [c * (c // 2) * 4, c // 2] + double(c, c // 2, c // 2)
        else:
            out += double(c, c // 2, c // 2 // (1 if k == 3 else 2))
    return out + [2 * b, 2]


def sections(case):
    """[(bits, indices into sizes(case))]: which tensors hold 8-bit moments and which hold 32-bit ones."""
    n = sizes(case)
    if case['op'] == 'clip':
        return [(0, list(range(len(n))))]
    small = [i for i, k in enumerate(n) if case['bits'] == 32 or k < MIN_8BIT]
    large = [i for i in range(len(n)) if i not in set(small)]
    return [(b, at) for b, at in ((8, large), (32, small)) if at]


def work(case):
    n, es = sizes(case), torch.empty(0, dtype=TYPES[case['dtype']]).element_size()
    total = sum(n)
    if case['op'] == 'clip':
        return {'bytes': 2 * es * total, 'flops': 3 * total}
    read_write = 0
    for bits, at in sections(case):
        k = sum(n[i] for i in at)
        read_write += k * (3 * es + 16) if bits == 32 else k * (3 * es + 4) + 4 * sum(-(-n[i] // BLOCK) for i in at)
    return {'bytes': read_write + 8 * len(n), 'flops': 15 * total}


# ---------------------------------------------------------------------------------------------------------- inputs
def _section(case, n, bits, gen):
    """Flat buffers of one section; each tensor of it is a view.  8-bit sections start every tensor on a block border,
    32-bit ones on 64 elements, the ragged list's without any padding."""
    pad = BLOCK if bits == 8 else 1 if case['kind'] == 'ragged' else 64
    starts, off = [], 0
    for k in n:
        starts.append(off)
        off += -(-k // pad) * pad
    dt, dev = TYPES[case['dtype']], 'cuda'
    counts = torch.tensor([b - a for a, b in zip(starts, starts[1:] + [off])], device=dev)
    used = torch.zeros(off, dtype=torch.bool, device=dev)
    for a, k in zip(starts, n):
        used[a:a + k] = True

    def rand():
        return torch.randn(off, generator=gen, device=dev) * used

    def spread(values):
        return torch.repeat_interleave(values, counts, output_size=off)

    # the layers' gradients lie orders of magnitude apart, a channel in eight is dead at this step
    t = len(n)
    mag = 10 ** (torch.rand(t, generator=gen, device=dev) * 2.0 - (2.5 if case['dtype'] == 'fp16' else 3.0))
    live = (torch.rand(-(-off // 64), generator=gen, device=dev) > 0.125).repeat_interleave(64)[:off]
    mag = spread(mag)
    s = dict(bits=bits, n=n, starts=starts, total=off, param=(0.05 * rand()).to(dt),
             grad=(mag * rand() * live).to(dt))
    if bits:
        age = torch.randint(1, 2 * case['age'] + 1, (t,), generator=gen, device=dev) if case['kind'] == 'ragged' else \
            torch.full((t,), case['age'], device=dev)
        if case['kind'] == 'ragged':
            age[::7] = 0                                  # tensors that join the training with this step
        s['step'] = age.float()
        old = spread((age > 0).float())
        m = 0.3 * mag * rand() * old
        v = (mag * (0.2 + rand().abs()) * old * used).square()
        if bits == 32:
            s['exp_avg'], s['exp_avg_sq'] = m, v
        else:
            s['exp_avg'], e_m = _nearest_codes(m, 0.0)
            s['exp_avg_root'], e_r = _nearest_codes(v.sqrt(), 2.0 ** -9)
            s['scales'] = torch.stack([e_m, e_r], 1).view(torch.float8_e8m0fnu)
        s['seed'] = 1234
        if not own:                                       # which tensor an element of the flat buffers belongs to
            s['owner'] = torch.repeat_interleave(torch.arange(t, device=dev), counts, output_size=off)
            s['position'] = torch.arange(off, device=dev) - spread(torch.cumsum(counts, 0) - counts)
    return s


def _nearest_codes(x, lowest):
    """Starting moments: codes rounded to nearest, scale bytes."""
    b = x.view(-1, BLOCK)
    e = _scale_byte(b.abs().amax(1))
    y = (b.double() * torch.exp2(127.0 - e.double())[:, None]).float()
    y = torch.where(y != 0, torch.sign(y) * y.abs().clamp(min=lowest), 0.0)
    return y.to(torch.float8_e4m3fn).view(-1), e.to(torch.uint8)


def _scale_byte(top):
    """127 + the smallest k >= -127 with top <= 448 * 2^k."""
    frac, power = torch.frexp(top.double())               # top = frac * 2^power, frac in [1/2, 1); 448 = 0.875 * 2^9
    return torch.where(top > 0, power - 9 + (frac > 0.875).int() + 127, 0).clamp(min=0)


def _views(s, name):
    return [s[name][a:a + k] for a, k in zip(s['starts'], s['n'])]


def prepare(case, seed):
    gen = torch.Generator(device='cuda')
    gen.manual_seed(int(seed))
    n = sizes(case)
    st = dict(case=case, limit=case['max_norm'], parts=[])
    st['parts'] = [_section(case, [n[i] for i in at], bits, gen) for bits, at in sections(case)]
    total = math.sqrt(sum(float(s['grad'].double().square().sum()) for s in st['parts']))
    if case['max_norm'] > 0 and total > 0:                # gradients that the limit cuts to a third
        for s in st['parts']:
            s['grad'].copy_(s['grad'].float() * (3.0 * case['max_norm'] / total))
    params = []
    for s in st['parts']:
        s['leaves'] = [torch.nn.Parameter(p) for p in _views(s, 'param')]
        for p, g in zip(s['leaves'], _views(s, 'grad')):
            p.grad = g
        params += s['leaves']
    st['params'] = params
    if own:
        root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), 'pytorch-unet_amd')
        if root not in sys.path:
            sys.path.insert(0, root)
        from unetk import optim
        st['optim'] = optim
        if case['op'] == 'adamw':
            opt = optim.AdamW(params, lr=case['lr'], betas=(0.9, case['beta2']), eps=1e-8, weight_decay=0.01,
                              max_norm=case['max_norm'] or None, state_bits=case['bits'], min_8bit_numel=MIN_8BIT,
                              seed=1234)
            for s in st['parts']:
                names = ('exp_avg', 'exp_avg_sq') if s['bits'] == 32 else ('exp_avg', 'exp_avg_root')
                moments = list(zip(*(_views(s, k) for k in names)))
                for i, p in enumerate(s['leaves']):
                    opt.state[p] = {'step': s['step'][i], names[0]: moments[i][0], names[1]: moments[i][1]}
                    if s['bits'] == 8:
                        a = s['starts'][i] // BLOCK
                        opt.state[p]['scales'] = s['scales'][a:a + -(-s['n'][i] // BLOCK)]
            st['opt'] = opt
    return st


# ---------------------------------------------------------------------------------------------------------- passes
def _outputs(st, norm):
    out = {} if norm is None else {'norm': norm}
    for s in st['parts']:
        for k in ('param', 'exp_avg', 'exp_avg_sq', 'exp_avg_root', 'scales', 'step'):
            if k in s and st['case']['op'] == 'adamw':
                out['%s.%d' % (k, s['bits'])] = s[k]
        if st['case']['op'] == 'clip':
            out['grad'] = s['grad']
    return out


def run(st):
    case = st['case']
    if case['op'] == 'clip':
        # every pass has something to cut: the limit falls from pass to pass
        st['limit'] *= 1.0 - 2.0 ** -12
        norm = st['optim'].clip_grad_norm_(st['params'], st['limit']) if own else _plain_clip(st)
        return _outputs(st, norm)
    if own:
        st['opt'].step()
        return _outputs(st, st['opt'].total_norm if case['max_norm'] else None)
    return _plain_step(st)


def _plain_norm(st):
    return sum(s['grad'].float().square().sum(dtype=torch.float64) for s in st['parts']).sqrt().float()


def _plain_clip(st):
    norm = _plain_norm(st)
    coef = (st['limit'] / (norm + 1e-6)).clamp(max=1.0)
    for s in st['parts']:
        s['grad'].copy_(s['grad'].float() * coef)
    return norm


def _plain_step(st):
    case = st['case']
    norm, coef = None, None
    if case['max_norm']:
        norm = _plain_norm(st)
        coef = (case['max_norm'] / (norm + 1e-6)).clamp(max=1.0)
    for s in st['parts']:
        _plain_section(s, case['lr'], 0.9, case['beta2'], 1e-8, 0.01, coef)
    return _outputs(st, norm)


def _plain_section(s, lr, b1, b2, eps, wd, coef):
    def spread(x):                                        # a tensor's value for each of its elements
        return x.index_select(0, s['owner'])

    s['step'] += 1
    t = s['step'].double()
    size = spread((lr / (1 - b1 ** t)).float())
    root2 = spread((1 - b2 ** t).sqrt().float())
    g = s['grad'].float()
    if coef is not None:
        g = g * coef
    if s['bits'] == 32:
        m = s['exp_avg'].mul_(b1).add_(g, alpha=1 - b1)
        r = s['exp_avg_sq'].mul_(b2).addcmul_(g, g, value=1 - b2).sqrt()
    else:
        scale = s['scales'].view(torch.uint8).double().sub(127).exp2().float().repeat_interleave(BLOCK, 0)
        m = (s['exp_avg'].float() * scale[:, 0]).mul_(b1).add_(g, alpha=1 - b1)
        r = (s['exp_avg_root'].float() * scale[:, 1]).square_().mul_(b2).addcmul_(g, g, value=1 - b2).sqrt_()
    s['param'].copy_(s['param'].float() * (1 - lr * wd) - size * m / (r / root2 + eps))
    if s['bits'] == 8:
        key = _mix((s['step'].long() * 0x9E3779B9 + s['seed']) & MASK)
        h = _mix(s['position'] ^ spread(key))
        e_m = _stochastic_codes(s['exp_avg'], m, h & 0xFFFF, 0.0)
        e_r = _stochastic_codes(s['exp_avg_root'], r, h >> 16, 2.0 ** -9)
        s['scales'].copy_(torch.stack([e_m, e_r], 1).to(torch.uint8).view(torch.float8_e8m0fnu))


def _mix(h):
    h = ((h ^ (h >> 16)) * 0x85EBCA6B) & MASK
    h = ((h ^ (h >> 13)) * 0xC2B2AE35) & MASK
    return h ^ (h >> 16)


def _stochastic_codes(out, x, u, lowest):
    """Rounds x to e4m3 codes of its block's scale, up with the probability of the distance; returns the scale bytes.
    `lowest`: what a value other than zero rounds to at least."""
    b = x.view(-1, BLOCK)
    e = _scale_byte(b.abs().amax(1))
    y = (b.double() * torch.exp2(127.0 - e.double())[:, None]).view(-1)
    ulp = torch.exp2((torch.frexp(y)[1].double() - 4).clamp(min=-9))
    q = torch.floor(y.abs() / ulp + (u.double() + 0.5) / 65536) * ulp
    q = torch.where(y != 0, q.clamp(min=lowest), 0.0)
    out.copy_((torch.sign(y) * q).float().to(torch.float8_e4m3fn))
    return e


# ------------------------------------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    """The step from its definition, tensor by tensor in 64 bits.  An 8-bit moment is given as the value that its code
    stands for before that is rounded to 8 bits."""
    st = prepare(case, seed)
    parts = st['parts']
    norm = math.sqrt(sum(float((s['grad'].double() ** 2).sum()) for s in parts))
    limit = st['limit'] * (1.0 - 2.0 ** -12) if case['op'] == 'clip' else case['max_norm']
    coef = min(1.0, limit / (norm + 1e-6)) if limit else 1.0
    out = {'norm': torch.tensor(norm, dtype=torch.float64)} if limit else {}
    if case['op'] == 'clip':
        return {**out, 'grad': parts[0]['grad'].double() * coef}
    b1, b2 = 0.9, case['beta2']
    for s in parts:
        bits = s['bits']
        param, m_out, r_out = (torch.zeros(s['total'], dtype=torch.float64, device='cuda') for _ in range(3))
        scales = torch.ones(s['total'] // BLOCK, 2, dtype=torch.float64, device='cuda') * 2.0 ** -127
        for i, (a, k) in enumerate(zip(s['starts'], s['n'])):
            t = float(s['step'][i]) + 1
            g = s['grad'][a:a + k].double() * coef
            m, v = s['exp_avg'][a:a + k].double(), s['exp_avg_sq' if bits == 32 else 'exp_avg_root'][a:a + k].double()
            blocks = slice(a // BLOCK, a // BLOCK + -(-k // BLOCK))
            if bits == 8:
                old = torch.exp2(s['scales'][blocks].view(torch.uint8).double() - 127).repeat_interleave(BLOCK, 0)[:k]
                m, v = m * old[:, 0], (v * old[:, 1]) ** 2
            m, v = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g ** 2
            p = s['param'][a:a + k].double() * (1 - case['lr'] * 0.01)
            param[a:a + k] = p - case['lr'] * (m / (1 - b1 ** t)) / ((v / (1 - b2 ** t)).sqrt() + 1e-8)
            for col, (x, to) in enumerate(((m, m_out), (v if bits == 32 else v.sqrt(), r_out))):
                if bits == 8:
                    x = torch.nn.functional.pad(x, (0, -k % BLOCK)).view(-1, BLOCK)
                    top = x.abs().amax(1).clamp(min=448 * 2.0 ** -127)
                    sc = torch.exp2(torch.ceil(torch.log2(top / 448)))
                    scales[blocks, col] = sc
                    x = (x / sc[:, None]).view(-1)[:k]
                to[a:a + k] = x
        out.update({'param.%d' % bits: param, 'exp_avg.%d' % bits: m_out, 'step.%d' % bits: s['step'].double() + 1,
                    ('exp_avg_sq.%d' if bits == 32 else 'exp_avg_root.%d') % bits: r_out})
        if bits == 8:
            out['scales.8'] = scales
    return out
