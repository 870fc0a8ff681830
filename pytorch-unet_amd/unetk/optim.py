"""clip_grad_norm_ + RMSprop as one fused pass over flat buffers.

The reference builds `optim.RMSprop(model.parameters(), lr, weight_decay=1e-8, momentum=0.999, foreach=True)`
(train.py:77-78) and each step runs `clip_grad_norm_(model.parameters(), 1.0)` then `optimizer.step()`
(train.py:115-116): about ten foreach passes over 31 M parameters.  Here the parameters are re-pointed (same
nn.Parameter objects, same state_dict) at views of ONE flat fp32 buffer laid out exactly like the flat gradient
buffer of unetk.ddp.FlatGrads, the optimizer state is two more flat buffers, and a step is two kernels
(include/unetk.h: unetk_clip_rmsprop_step).  Subclasses torch.optim.Optimizer so LR schedulers
(train.py:79 ReduceLROnPlateau) keep working through param_groups[0]['lr'].

`AdamW` and `clip_grad_norm_` are the same step for other users' needs: any list of parameter tensors wherever they lie
(or the flat buffers above), decoupled weight decay, moments in 32 or in 8 bits, the clip in front of the step or by itself.
"""
import contextlib
import copy
import weakref
from array import array
from itertools import chain
from operator import is_

import torch

from . import _native as nat
from ._native import check, dtype_code, fn, stream_ptr
from .blocks import wrote_in_place


class ClipRMSprop(torch.optim.Optimizer):
    def __init__(self, flat_grads, lr=1e-2, alpha=0.99, eps=1e-8, weight_decay=0.0, momentum=0.0, max_norm=None):
        self.fg = flat_grads
        super().__init__(flat_grads.params, dict(lr=lr, alpha=alpha, eps=eps, weight_decay=weight_decay,
                                                 momentum=momentum, max_norm=max_norm))
        self.pflat = self.square_avg = self.momentum_buf = None
        self.total_norm = None          # device fp64 scalar: ||grad||_2 before clipping (clip_grad_norm_'s result)
        self._steps = 0
        self._flatten()

    def zero_grad(self, set_to_none=True):
        """train.py:113.  The flat gradient buffer is rewritten by every backward pass, so there is nothing to zero;
        the call discards the previous pass's gradients, so that a step() before the next pass does not apply them again (a
        backward without it or step() in between would be gradient accumulation, which the flat buffer does not do:
        FlatGrads.initial_grads raises)."""
        self.fg.discard(set_to_none)
        super().zero_grad(set_to_none=set_to_none)

    # ---- checkpoint / resume in torch.optim.RMSprop's own format (train.py saves only the model's state_dict, but a
    # user who checkpoints the optimizer can move between the two, in BOTH directions): per-parameter 'step',
    # 'square_avg', 'momentum_buffer', keyed by the parameter's index in net.parameters() order -- the order a stock
    # optimizer built from `net.parameters()` maps indices by (it checks group sizes only, not shapes)
    def state_dict(self):
        g = self.param_groups[0]
        order = list(self.fg.module_order)
        group = {k: v for k, v in g.items() if k != 'params'}
        group.update(centered=False, params=list(range(len(order))), unetk_order='module')
        state = {}
        if self._steps > 0:
            for i, p in enumerate(order):
                off, n = self.fg.offsets[id(p)], p.numel()
                st = {'step': torch.tensor(float(self._steps)),
                      'square_avg': self.square_avg[off:off + n].view(p.shape).clone()}
                if g['momentum'] > 0:
                    st['momentum_buffer'] = self.momentum_buf[off:off + n].view(p.shape).clone()
                state[i] = st
        return {'state': state, 'param_groups': [group]}

    def load_state_dict(self, state_dict):
        groups = state_dict['param_groups']
        if len(groups) != 1 or len(groups[0]['params']) != len(self.fg.params):
            raise ValueError('ClipRMSprop.load_state_dict: expected one parameter group over the same parameters')
        if groups[0].get('centered', False):
            raise ValueError('ClipRMSprop.load_state_dict: centered RMSprop state cannot be loaded')
        g = self.param_groups[0]
        for k in ('lr', 'alpha', 'eps', 'weight_decay', 'momentum', 'max_norm'):
            if k in groups[0]:
                g[k] = groups[0][k]
        self.square_avg.zero_()
        self.momentum_buf.zero_()
        steps = 0
        order = self._saved_order(groups[0])
        for i, st in state_dict['state'].items():
            p = order[int(i)]
            off, n = self.fg.offsets[id(p)], p.numel()
            if tuple(st['square_avg'].shape) != tuple(p.shape):
                raise ValueError('ClipRMSprop.load_state_dict: state shape does not match the parameter')
            self.square_avg[off:off + n].view(p.shape).copy_(st['square_avg'])
            if 'momentum_buffer' in st and st['momentum_buffer'] is not None:
                self.momentum_buf[off:off + n].view(p.shape).copy_(st['momentum_buffer'])
            steps = max(steps, int(float(st.get('step', 0))))
        self._steps = steps

    def _saved_order(self, group):
        """Checkpoints of a stock torch.optim.RMSprop and of this class (marker `unetk_order`) number the parameters in
        net.parameters() order; files this class wrote before it carried the marker (round 2: 'max_norm' present, no
        marker) used gradient-completion order and still load."""
        if 'max_norm' in group and group.get('unetk_order') != 'module':
            return self.fg.params
        return list(self.fg.module_order)

    def _flatten(self):
        """(Re-)point every parameter at its slice of one flat buffer; optimizer state survives a re-flatten."""
        fg = self.fg
        dev = fg.params[0].device
        if dev.type != 'cuda':
            raise RuntimeError('ClipRMSprop runs on the MI355X kernels: parameters must be on a cuda device')
        pflat = torch.zeros(fg.total, dtype=torch.float32, device=dev)
        for p in fg.params:
            if p.dtype != torch.float32:
                raise RuntimeError('ClipRMSprop: parameters must be fp32 (the reference keeps fp32 master weights)')
            off = fg.offsets[id(p)]
            view = pflat[off:off + p.numel()].view(p.shape)
            view.copy_(p.data)
            p.data = view
        self.pflat = pflat
        if self.square_avg is None:
            self.square_avg = torch.zeros_like(pflat)
            self.momentum_buf = torch.zeros_like(pflat)
            self._ws = torch.empty(int(fn['unetk_clip_rmsprop_workspace_bytes']()), dtype=torch.uint8, device=dev)
            self.total_norm = torch.zeros((), dtype=torch.float64, device=dev)

    def _still_flat(self):
        base = self.pflat.data_ptr()
        return all(p.data_ptr() == base + 4 * self.fg.offsets[id(p)] for p in self.fg.params)

    @torch.no_grad()
    def step(self, closure=None):
        if closure is not None:
            raise RuntimeError('ClipRMSprop.step takes no closure')
        grads = self.fg.flat
        if grads is None:
            raise RuntimeError('ClipRMSprop.step: no gradients (run backward through the UNet first)')
        if not self._still_flat():           # e.g. net.to(memory_format=...) after construction re-allocated them
            self._flatten()
        g = self.param_groups[0]
        max_norm = g['max_norm'] if g['max_norm'] is not None else 0.0
        check(fn['unetk_clip_rmsprop_step'](self.pflat.data_ptr(), grads.data_ptr(), self.square_avg.data_ptr(),
                                            self.momentum_buf.data_ptr(), self.fg.total, self._ws.data_ptr(),
                                            self._ws.numel(), self.total_norm.data_ptr(), float(max_norm),
                                            float(g['lr']), float(g['alpha']), float(g['eps']),
                                            float(g['weight_decay']), float(g['momentum']), stream_ptr()),
              'unetk_clip_rmsprop_step')
        wrote_in_place(self.fg.params, stream_ptr())
        self._steps += 1
        self.fg.consume()
        return None


# ---------------------------------------------------------------------------------------- many tensors at once
BLOCK = 256                     # elements that share one scale per moment (unetk_adamw_update)
_CODE, _SCALE = torch.float8_e4m3fn, torch.float8_e8m0fnu
_TYPES = {torch.float32, torch.bfloat16, torch.float16}

# one C call per tensor each: a step of small tensors is bound by what the host asks of them
_get_pointer, _get_numel, _get_device = torch.Tensor.data_ptr, torch.Tensor.numel, torch.Tensor.get_device
_get_contiguous, _get_dtype, _get_stride = torch.Tensor.is_contiguous, torch.Tensor.dtype.__get__, torch.Tensor.stride
_get_shape, _get_nbytes = torch.Tensor.shape.__get__, torch.Tensor.nbytes.__get__
_get_wanted = torch.Tensor.requires_grad.__get__


def _address(words):
    return words.buffer_info()[0]


def _on_device(device):
    """Launches go to the tensors' device whatever the current one is, on that device's current stream."""
    if device.type != 'cuda' or torch.cuda.current_device() == device.index:
        return contextlib.nullcontext()
    return torch.cuda.device(device)


def _is_dense(t):
    """Whether the elements fill one piece of memory, in any order of the dimensions."""
    if t.is_contiguous():
        return True
    expect = 1
    for stride, size in sorted((st, n) for st, n in zip(t.stride(), t.shape) if n != 1):
        if stride != expect:
            return False
        expect *= size
    return True


def _require(t, what, owner='AdamW'):
    if t.layout != torch.strided:
        raise RuntimeError(f'{owner}: {what} must be strided tensors, got {t.layout}')
    if not t.is_cuda:
        raise RuntimeError(f'{owner} runs on the MI355X kernels: {what} must be on a cuda device (no CPU fallback)')
    dtype_code(t.dtype)
    if not _is_dense(t):
        raise RuntimeError(f'{owner}: {what} must be dense (no gaps, no overlaps), got strides {t.stride()} for shape '
                           f'{tuple(t.shape)}')


def _memory_order(t):
    """The elements of a dense tensor as they lie in memory, as one dimension."""
    return t.view(-1) if t.is_contiguous() else t.as_strided((t.numel(),), (1,))


def clip_grad_norm_(parameters, max_norm, norm_type=2.0, error_if_nonfinite=False, foreach=None):
    """torch.nn.utils.clip_grad_norm_ (reference train.py:115) over any list of tensors in two passes: the 2-norm of all
    gradients together, then every gradient times min(1, max_norm / (norm + 1e-6)) in place.  Gradients may be fp32, bf16 and
    fp16 mixed; the sum of squares is taken in fp64.  Nothing is written where the norm is within the limit.  Returns the norm
    as an fp32 scalar on the device; reads nothing back unless `error_if_nonfinite`.  `foreach` is accepted and ignored."""
    if isinstance(parameters, torch.Tensor):
        parameters = [parameters]
    if float(norm_type) != 2.0:
        raise ValueError('clip_grad_norm_: only the 2-norm is implemented')
    max_norm = float(max_norm)
    if not max_norm >= 0:
        raise ValueError(f'clip_grad_norm_: max_norm must not be negative, got {max_norm}')
    grads = [g for g in [p.grad for p in parameters] if g is not None]
    if not grads:
        return torch.tensor(0.0)
    if len(set(map(id, grads))) != len(grads):
        raise ValueError('clip_grad_norm_: a parameter appears twice')
    if len(set(map(_get_device, grads))) != 1:
        raise RuntimeError('clip_grad_norm_: gradients must be on one device')
    types = dict.fromkeys(map(_get_dtype, grads))        # in their order: the norm is summed in it
    if not grads[0].is_cuda or not types.keys() <= _TYPES or not all(map(_get_contiguous, grads)):
        for g in grads:
            _require(g, 'gradients', 'clip_grad_norm_')
    sets = [(dtype_code(t), grads if len(types) == 1 else [g for g in grads if g.dtype == t]) for t in types]
    device = grads[0].device
    with _on_device(device):
        stream = stream_ptr()
        sets = [(code, len(gs), array('q', map(_get_pointer, gs)), array('q', map(_get_numel, gs))) for code, gs in sets]
        partials = torch.empty(sum(fn['unetk_grad_partials'](n) for _, n, _, _ in sets), dtype=torch.float64, device=device)
        norm = torch.empty((), dtype=torch.float32, device=device)
        at, count = partials.data_ptr(), 0
        for code, n, pointers, numel in sets:
            written = fn['unetk_grad_sumsq'](_address(pointers), _address(numel), n, code, at + 8 * count, stream)
            if written == nat.ERR_ARG:                   # all else that it refuses was looked at above
                raise RuntimeError('clip_grad_norm_: gradients must not overlap in memory')
            count += _written(written, 'unetk_grad_sumsq')
        if error_if_nonfinite:
            # the very norm that is returned and divided by (fp32: infinite where the sum in fp64 is not), before anything is scaled
            zero = array('q', [0])
            check(fn['unetk_grad_clip'](_address(zero), _address(zero), 1, sets[0][0], at, count, max_norm, norm.data_ptr(), stream),
                  'unetk_grad_clip')
            if not bool(torch.isfinite(norm)):
                raise RuntimeError('clip_grad_norm_: the norm of the gradients is not finite, so they cannot be clipped')
        for code, n, pointers, numel in sets:
            check(fn['unetk_grad_clip'](_address(pointers), _address(numel), n, code, at, count, max_norm, norm.data_ptr(),
                                        stream), 'unetk_grad_clip')
    torch.autograd.graph.increment_version(grads)
    return norm


def _not_captured(what):
    if torch.cuda.is_current_stream_capturing():
        raise RuntimeError(f'AdamW: take one step before capturing: a graph cannot {what}, every replay would do it again')


def _written(count, what):
    if count < 0:
        check(int(count), what)
    return int(count)


def dequantize_moment(codes, scales):
    """fp32 values, in memory order, of 8-bit codes and their block's scales (one column of a state's `scales`)."""
    x = _memory_order(codes).to(torch.float32)
    scale = torch.ldexp(torch.ones((), device=x.device), scales.contiguous().view(torch.uint8).to(torch.int32) - 127)
    return x * scale.repeat_interleave(BLOCK)[:x.numel()]


def quantize_moment(x, keep_positive=False):
    """Codes (to nearest) and scales of fp32 values that lie in one dimension.  `keep_positive`: what is not zero does not
    become zero, as a root of a second moment must not."""
    n = x.numel()
    b = torch.nn.functional.pad(x.detach().to(torch.float32), (0, -n % BLOCK)).view(-1, BLOCK)
    finite = torch.where(torch.isfinite(b), b, 0.0)
    frac, power = torch.frexp(finite.abs().amax(1))                 # top = frac * 2^power; 448 = 0.875 * 2^9
    byte = torch.where(frac > 0, power + (frac > 0.875).to(torch.int32) + 118, 0).clamp(min=0)
    y = b.double() * torch.exp2(127.0 - byte.double())[:, None]
    if keep_positive:
        y = torch.where(y != 0, torch.sign(y) * y.abs().clamp(min=2.0 ** -9), y)
    y = torch.where(torch.isfinite(y), y, float('nan')).to(torch.float32).to(_CODE)
    return y.view(-1)[:n], byte.to(torch.uint8).view(_SCALE)


class AdamW(torch.optim.Optimizer):
    """AdamW over any list of parameters, the whole step in two launches per 64 tensors of one type (include/unetk.h:
    unetk_adamw_prepare, unetk_adamw_update), with clip_grad_norm_(max_norm) over all of them in front.

    params: an iterable of tensors or of parameter groups, on one GPU, in fp32, bf16 or fp16; or a unetk.ddp.FlatGrads, whose
    flat gradient buffer is then read in place.  Any dense memory layout; a gradient that is laid out unlike its parameter is
    copied first.
    max_norm: limit of the 2-norm of all gradients together (one value for all groups), None for no clip.  The gradients
    themselves stay as they are; `total_norm` holds the norm before the clip (fp32, on the device) after a step, zero if there
    were none.
    state_bits: 32 keeps `exp_avg` and `exp_avg_sq` in fp32 whatever the parameter's type.  8 keeps them as fp8 codes with a
    power-of-two scale per 256 elements (2.02 instead of 8 bytes a parameter), rounded stochastically from `seed`, the step and the
    element's index, for tensors of at least `min_8bit_numel` elements; smaller ones (biases, BatchNorm) keep 32 bits.
    eps is then 0 or at least 2^-126.
    lr: a float, or an fp32 scalar tensor on the device, which a captured graph reads anew at each replay.

    Parameters, moments and step counts that overlap in memory are refused: they would be written in any order.
    The rounding is the same on every rank of a data-parallel job.  A parameter that is laid out anew (net.to(memory_format=...))
    takes its moments along, 8-bit ones rounded to nearest in their new blocks.
    state[p]: `step` (fp32 scalar on the device), `exp_avg`, and `exp_avg_sq` or, in 8 bits, `exp_avg_root` (the square root)
    and `scales`.  With 32 bits state_dict() is torch.optim.AdamW's; load_state_dict() takes that one's and either form.
    Under torch.amp.GradScaler the step is skipped on the device, without a read-back.  A step can be captured into a graph once
    the state exists (after a first step, or a load_state_dict).
    """
    _step_supports_amp_scaling = True

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, max_norm=None, state_bits=32,
                 min_8bit_numel=4096, seed=0):
        self.fg = params if hasattr(params, 'module_order') else None
        if state_bits not in (8, 32):
            raise ValueError(f'AdamW: state_bits must be 8 or 32, got {state_bits}')
        self.state_bits, self.min_8bit_numel, self.seed = state_bits, int(min_8bit_numel), int(seed) & 0xFFFFFFFF
        self.total_norm = None
        self._plan = self._apart = None
        if self.fg is not None:          # net.parameters() order, as a stock optimizer numbers its state
            params = [p for p in self.fg.module_order if id(p) in self.fg.offsets]
            for p in params:             # laid out like its view of the flat gradients
                p.data = p.data.contiguous()
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, max_norm=max_norm))

    def add_param_group(self, group):
        super().add_param_group(group)
        self._plan = None
        try:
            self._check_group(self.param_groups[-1])
        except Exception:
            self.param_groups.pop()
            raise

    def _check_group(self, g):
        if len({id(p) for p in g['params']}) != len(g['params']):
            raise ValueError('AdamW: a parameter appears twice')
        self._check_hyperparameters(g, [g, self.param_groups[0]])
        if self.fg is not None and not all(id(p) in self.fg.offsets for p in g['params']):
            raise ValueError('AdamW: a parameter has no place in the flat gradient buffer')
        for p in g['params']:
            _require(p, 'parameters')
            if p.device != next(q for h in self.param_groups for q in h['params']).device:
                raise RuntimeError('AdamW: parameters must be on one device')

    def _check_hyperparameters(self, g, groups):
        for k in ('lr', 'eps', 'weight_decay'):
            if not isinstance(g[k], torch.Tensor) and not g[k] >= 0:
                raise ValueError(f'AdamW: {k} must not be negative, got {g[k]}')
        if not all(0.0 <= b < 1.0 for b in g['betas']):
            raise ValueError(f"AdamW: betas must lie in [0, 1), got {g['betas']}")
        _usable_eps(g, self.state_bits)
        _common_max_norm(groups)

    def __getstate__(self):
        return {**super().__getstate__(), 'fg': self.fg, 'state_bits': self.state_bits, 'min_8bit_numel': self.min_8bit_numel,
                'seed': self.seed, 'total_norm': self.total_norm}

    def __setstate__(self, state):
        super().__setstate__(state)
        self._plan = self._apart = None

    def zero_grad(self, set_to_none=True):
        if self.fg is not None:
            self.fg.discard(set_to_none)
        super().zero_grad(set_to_none=set_to_none)

    # ---- state
    def _new_state(self, p):
        _not_captured('make its state')
        st = {'step': torch.zeros((), dtype=torch.float32, device=p.device)}
        if self.state_bits == 8 and p.numel() >= self.min_8bit_numel:
            for k in ('exp_avg', 'exp_avg_root'):
                st[k] = torch.zeros_like(p, dtype=torch.uint8).view(_CODE)
            st['scales'] = torch.zeros(-(-p.numel() // BLOCK), 2, dtype=torch.uint8, device=p.device).view(_SCALE)
        else:
            for k in ('exp_avg', 'exp_avg_sq'):
                st[k] = torch.zeros_like(p, dtype=torch.float32)
        return st

    def _check_state(self, p, st):
        """The moments lie as the parameter does; moves them if the parameter was laid out anew (net.to(memory_format=...))."""
        bits = 8 if 'scales' in st else 32
        names = ('exp_avg', 'exp_avg_root') if bits == 8 else ('exp_avg', 'exp_avg_sq')
        want = _CODE if bits == 8 else torch.float32
        for k in names:
            t = st[k]
            if t.dtype != want or t.shape != p.shape or t.device != p.device:
                raise RuntimeError(f'AdamW: state {k!r} must be {want} of shape {tuple(p.shape)} on {p.device}')
        step = st['step']
        if not torch.is_tensor(step) or step.dtype != torch.float32 or step.device != p.device or step.numel() != 1:
            raise RuntimeError("AdamW: state 'step' must be an fp32 scalar on the parameter's device")
        if bits == 8:
            sc = st['scales']
            if sc.dtype != _SCALE or tuple(sc.shape) != (-(-p.numel() // BLOCK), 2) or not sc.is_contiguous() or \
                    sc.device != p.device:
                raise RuntimeError("AdamW: state 'scales' must be contiguous float8_e8m0fnu [ceil(numel / 256), 2]")
        if any(st[k].stride() != p.stride() for k in names):
            _not_captured('lay its state out anew')
            st.update(_fit_moments(p, st, bits))
        return bits

    # ---- checkpoint / resume.  The file's form (32-bit as torch.optim.AdamW writes it, or 8-bit) need not be this one's.
    def load_state_dict(self, state_dict):
        state_dict = dict(state_dict)                    # a hook may exchange entries
        for hook in list(self._optimizer_load_state_dict_pre_hooks.values()):
            changed = hook(self, state_dict)
            state_dict = state_dict if changed is None else changed
        groups = state_dict['param_groups']
        if [len(g['params']) for g in groups] != [len(g['params']) for g in self.param_groups]:
            raise ValueError('AdamW.load_state_dict: expected the same parameter groups')
        for g in groups:
            if g.get('amsgrad') or g.get('maximize'):
                raise ValueError('AdamW.load_state_dict: amsgrad and maximize are not implemented')
        params = [p for g in self.param_groups for p in g['params']]
        state = {}
        for index, p in zip([i for g in groups for i in g['params']], params):
            if index not in state_dict['state']:
                continue
            st = state_dict['state'][index]
            if not {'step', 'exp_avg', *(('exp_avg_root',) if 'scales' in st else ('exp_avg_sq',))} <= set(st):
                raise ValueError('AdamW.load_state_dict: not the state of an AdamW')
            second = 'exp_avg_root' if 'scales' in st else 'exp_avg_sq'
            if any(tuple(st[k].shape) != tuple(p.shape) for k in ('exp_avg', second)):
                raise ValueError('AdamW.load_state_dict: state shape does not match the parameter')
            if 'scales' in st and (any(st[k].dtype != _CODE for k in ('exp_avg', second)) or st['scales'].dtype != _SCALE
                                   or tuple(st['scales'].shape) != (-(-p.numel() // BLOCK), 2)):
                raise ValueError('AdamW.load_state_dict: 8-bit moments must be float8_e4m3fn with float8_e8m0fnu scales of shape '
                                 '[ceil(numel / 256), 2]')
            bits = 8 if self.state_bits == 8 and p.numel() >= self.min_8bit_numel else 32
            state[p] = _fit_moments(p, st, bits)
            state[p]['step'] = torch.tensor(float(st['step']), dtype=torch.float32, device=p.device)
        # a group takes over all that the file's holds (a scheduler's entries too) and keeps what the file's lacks
        merged = [{**own, **{k: copy.deepcopy(v) for k, v in g.items() if k != 'params'}, 'lr': float(g['lr'])}
                  for own, g in zip(self.param_groups, groups)]
        for g in merged:
            self._check_hyperparameters(g, merged)
        for own, g in zip(self.param_groups, merged):
            if isinstance(own['lr'], torch.Tensor):      # a captured graph reads this very tensor
                g['lr'] = own['lr'].fill_(g['lr'])
            own.update(g)
        self._plan = None
        self.state.clear()
        self.state.update(state)
        for hook in list(self._optimizer_load_state_dict_post_hooks.values()):
            hook(self)

    # ---- step
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        if self.fg is not None and self.fg.flat is None:
            raise RuntimeError('AdamW.step: no gradients (run backward through the UNet first)')
        plan = self._plan
        pointers = plan.pointers(self) if plan is not None else None
        device = next((p.device for g in self.param_groups for p in g['params']), torch.device('cpu'))
        with _on_device(device):
            if pointers is None:                         # the first step, or something moved, came or went
                plan = self._plan = None
                with torch.no_grad():
                    plan, pointers, copies = self._make_plan()
            if plan.params:
                stream = stream_ptr()
                self._launch(plan, pointers, stream)
                wrote_in_place(plan.params, stream)
            else:                                        # no gradients: a norm of zero, not an earlier step's
                limit = _common_max_norm(self.param_groups)
                self.total_norm = None if limit is None else torch.zeros((), dtype=torch.float32, device=device)
        self._plan = plan
        if self.fg is not None:
            self.fg.consume()
        return loss

    def _make_plan(self):
        """Looks every tensor over: the plan of this step, the gradients' pointers, and copies of gradients that lie unlike their
        parameters (to be kept until the launch)."""
        rows, absent, copies, state = [], [], [], self.state
        for at, group in enumerate(self.param_groups):
            for p in group['params']:
                # the flat buffer has room for frozen parameters too
                g = p.grad if self.fg is None else self.fg.views.get(p) if p.requires_grad else None
                if g is None:
                    absent.append(p)
                    continue
                if self.fg is not None and not p.is_contiguous():
                    _not_captured('lay its parameters out anew')
                    p.data = p.data.contiguous()
                st = state.get(p)
                if not st:
                    _require(p, 'parameters')
                    st = state[p] = self._new_state(p)
                rows.append((at, p, st, g))
        if rows and not _all_usual(rows):
            for k, (at, p, st, g) in enumerate(rows):
                _require(p, 'parameters')
                self._check_state(p, st)
                if g.layout != torch.strided or g.dtype != p.dtype or g.device != p.device or g.shape != p.shape:
                    raise RuntimeError("AdamW: a gradient must be a strided tensor of its parameter's type, shape and device")
                if g.stride() != p.stride():
                    copies.append(torch.empty_like(p).copy_(g))
                    rows[k] = at, p, st, copies[-1]
        sets = {}
        for at, p, st, g in rows:
            sets.setdefault((at, p.dtype), []).append((p, st, g))
        return _Plan(self, sets, absent), array('q', [g.data_ptr() for rs in sets.values() for _, _, g in rs]), copies

    def _launch(self, plan, pointers, stream):
        device = plan.device
        # all that can be wrong with the groups is found here: once a launch has counted, the step has to go through
        hyper = [_hyperparameters(self.param_groups[at], device, self.state_bits) for at, _, _, _, _ in plan.sets]
        max_norm = _common_max_norm(self.param_groups)
        grad_scale, found_inf = getattr(self, 'grad_scale', None), getattr(self, 'found_inf', None)
        for t in (grad_scale, found_inf):
            if t is not None and (t.dtype != torch.float32 or t.device != device or t.numel() != 1):
                raise RuntimeError("AdamW: grad_scale and found_inf must be fp32 scalars on the parameters' device")
        scale_ptr = grad_scale.data_ptr() if grad_scale is not None else None
        found_ptr = found_inf.data_ptr() if found_inf is not None else None
        # scratch of this call alone, from the allocator of the stream it runs on: calls share none of it
        scratch = torch.empty(plan.words[max_norm is not None], dtype=torch.float64, device=device)
        coefs, partials, norm_ptr, count = scratch.data_ptr(), None, None, 0
        self.total_norm = None
        if max_norm is not None:
            self.total_norm = torch.empty((), dtype=torch.float32, device=device)
            partials, norm_ptr = coefs + 16 * len(plan.params), self.total_norm.data_ptr()
        grads = _address(pointers)
        for (_, code, first, n, table), (lr, lr_ptr, beta1, beta2, _, weight_decay) in zip(plan.sets, hyper):
            count += _written(fn['unetk_adamw_prepare'](table, grads + 8 * first, n, code, lr, lr_ptr, beta1, beta2, weight_decay,
                                                        self.seed, found_ptr, coefs + 16 * first,
                                                        partials + 8 * count if partials else None, stream),
                              'unetk_adamw_prepare')
        for (_, code, first, n, table), (_, _, beta1, beta2, eps, _) in zip(plan.sets, hyper):
            check(fn['unetk_adamw_update'](table, grads + 8 * first, n, code, beta1, beta2, eps, scale_ptr, found_ptr,
                                           coefs + 16 * first, partials, count, max_norm or 0.0, norm_ptr, stream),
                  'unetk_adamw_update')


def _common_max_norm(groups):
    """The one limit of all groups, as a float or None."""
    max_norm = groups[0]['max_norm']
    if max_norm is not None:
        max_norm = float(max_norm)
        if not max_norm > 0:
            raise ValueError(f'AdamW: max_norm must be positive or None, got {max_norm}')
    if len(groups) > 1 and any(g['max_norm'] != max_norm for g in groups):
        raise ValueError('AdamW: the clip is over all groups: max_norm must be the same in each')
    return max_norm


def _usable_eps(group, bits):
    """The 8-bit update takes a reciprocal whose argument must not be subnormal."""
    eps = float(group['eps'])
    if bits == 8 and 0.0 < eps < 2.0 ** -126:
        raise ValueError(f'AdamW: with 8-bit moments eps must be 0 or at least 2^-126, got {eps}')
    return eps


def _hyperparameters(group, device, bits):
    """(lr, pointer to an lr on the device or None, beta1, beta2, eps, weight_decay) as a launch takes them."""
    lr, lr_ptr = group['lr'], None
    if isinstance(lr, torch.Tensor) and lr.is_cuda:
        if lr.dtype != torch.float32 or lr.device != device or lr.numel() != 1:
            raise RuntimeError("AdamW: a tensor lr must be an fp32 scalar on the parameters' device")
        lr, lr_ptr = 0.0, lr.data_ptr()
    beta1, beta2 = group['betas']
    return float(lr), lr_ptr, float(beta1), float(beta2), _usable_eps(group, bits), float(group['weight_decay'])


def _all_usual(rows):
    """What nearly every step finds, looked at attribute by attribute for all tensors together: everything contiguous, of the
    right types and shapes, on one device.  False leaves it to the checks of each tensor, which say what is wrong."""
    _, params, states, grads = zip(*rows)
    try:
        wide = [(p, st) for p, st in zip(params, states) if 'scales' not in st]
        code = [(p, st) for p, st in zip(params, states) if 'scales' in st]
        like = list(params) * 3
        moments = [st['exp_avg'] for st in states] + [st['exp_avg_root' if 'scales' in st else 'exp_avg_sq'] for st in states]
        steps, scales = [st['step'] for st in states], [st['scales'] for _, st in code]
        every = [*params, *grads, *moments, *scales]
        return (all(map(_get_contiguous, every))
                and len(set(map(_get_device, [*every, *steps]))) == 1 and params[0].is_cuda
                and list(map(_get_dtype, params)) == list(map(_get_dtype, grads)) and set(map(_get_dtype, params)) <= _TYPES
                and list(map(_get_shape, like)) == list(map(_get_shape, [*grads, *moments]))
                and {st[k].dtype for _, st in wide for k in ('exp_avg', 'exp_avg_sq')} <= {torch.float32}
                and {st[k].dtype for _, st in code for k in ('exp_avg', 'exp_avg_root')} <= {_CODE}
                and set(map(_get_dtype, steps)) == {torch.float32} and set(map(_get_numel, steps)) == {1}
                and set(map(_get_dtype, scales)) <= {_SCALE}
                and all(tuple(st['scales'].shape) == (-(-p.numel() // BLOCK), 2) for p, st in code))
    except (KeyError, AttributeError, TypeError, RuntimeError):
        return False


class _Plan:
    """The launch tables of an optimizer's own parameters and moments: where they lie, no value of theirs; gradients are looked up
    at every step.  What one step found out serves the next as long as nothing moved, came or went.  It does not keep the state
    alive, neither its tensors nor the dictionaries that hold them (a user may move it off the device or drop it between steps):
    weak references tell whether a tensor is the same one, its address whether it is where it was."""

    def __init__(self, opt, sets, absent):
        rows = [r for rs in sets.values() for r in rs]
        self.params, self.absent = [p for p, _, _ in rows], absent
        self.device = rows[0][0].device if rows else None
        self.every = [list(g['params']) for g in opt.param_groups]
        self.sets, self.tables, first = [], [], 0
        for (at, dtype), rs in sets.items():
            table = array('q', [w for p, st, _ in rs for w in
                                (p.data_ptr(), st['exp_avg'].data_ptr(),
                                 st['exp_avg_root' if 'scales' in st else 'exp_avg_sq'].data_ptr(),
                                 st['scales'].data_ptr() if 'scales' in st else 0, st['step'].data_ptr(), p.numel())])
            self.tables.append(table)
            self.sets.append((at, dtype_code(dtype), first, len(rs), _address(table)))
            first += len(rs)
        self._check_apart(opt)
        self.words = [2 * first, 2 * first + sum(int(fn['unetk_grad_partials'](s[3])) for s in self.sets)]
        self.owners = list(opt.state)
        tensors = list(chain.from_iterable(map(dict.values, opt.state.values())))
        self.usable = all(map(torch.is_tensor, tensors))      # a user may keep other things there: then every step looks anew
        if not self.usable:
            return
        self.ids, self.gone = list(map(id, tensors)), []
        self.refs = [weakref.ref(t, self.gone.append) for t in tensors]          # an id is its tensor's while that lives
        self.where = list(map(_get_pointer, self.params)) + list(map(_get_pointer, tensors))
        # a parameter or gradient that became smaller where it lies must not be stepped with the old table: bytes tell, but not
        # one 16-bit type from the other
        self.nbytes, types = list(map(_get_nbytes, self.params)), list(map(_get_dtype, self.params))
        self.types = types if set(types) - {torch.float32} else None
        self.contiguous = all(map(_get_contiguous, self.params))
        self.strides = None if self.contiguous else list(map(_get_stride, self.params))
        if opt.fg is not None:
            self.offsets = [4 * opt.fg.offsets[id(p)] for p in self.params]

    def _check_apart(self, opt):
        """What a step writes must not overlap: the workgroups of a launch come to it in any order."""
        layout = [(code, table.tobytes()) for (_, code, _, _, _), table in zip(self.sets, self.tables)]
        if not layout or layout == opt._apart:           # looked at when the tensors last came to lie so
            return
        rows, size = array('q'), array('B')
        for (_, code, _, n, _), table in zip(self.sets, self.tables):
            rows.extend(table)
            size.extend([4 if code == nat.F32 else 2] * n)
        if _written(fn['unetk_adamw_overlaps'](_address(rows), _address(size), len(size)), 'unetk_adamw_overlaps'):
            raise RuntimeError('AdamW: parameters, moments and step counts must not overlap in memory')
        opt._apart = layout

    def pointers(self, opt):
        """The gradients' pointers if the plan holds for this step, else None."""
        params, groups = self.params, opt.param_groups
        if not self.usable or len(groups) != len(self.every):
            return None
        for group, had in zip(groups, self.every):
            if len(group['params']) != len(had) or not all(map(is_, group['params'], had)):
                return None
        if len(opt.state) != len(self.owners) or not all(map(is_, opt.state, self.owners)):
            return None
        tensors = list(chain.from_iterable(map(dict.values, opt.state.values())))
        if self.gone or list(map(id, tensors)) != self.ids or \
                list(map(_get_pointer, params)) + list(map(_get_pointer, tensors)) != self.where or \
                list(map(_get_nbytes, params)) != self.nbytes:
            return None
        if not all(map(_get_contiguous, params)) if self.contiguous else list(map(_get_stride, params)) != self.strides:
            return None
        if opt.fg is not None:
            if not all(map(_get_wanted, params)) or any(map(_get_wanted, self.absent)):
                return None
            base = opt.fg.flat.data_ptr()
            return array('q', [base + o for o in self.offsets])
        grads = [p.grad for p in params]
        if any(p.grad is not None for p in self.absent):
            return None
        try:
            if list(map(_get_nbytes, grads)) != self.nbytes or self.types and list(map(_get_dtype, grads)) != self.types:
                return None
            if not all(map(_get_contiguous, grads)) if self.contiguous else list(map(_get_stride, grads)) != self.strides:
                return None
            return array('q', list(map(_get_pointer, grads)))
        except (TypeError, RuntimeError):                # a gradient that is None, or not a strided tensor
            return None


def _fit_moments(p, st, bits):
    """The moments of a state in the form and memory layout that parameter `p` needs."""
    if bits == 8 and 'scales' in st and st['exp_avg'].stride() == p.stride():
        return {k: st[k].view(torch.uint8).to(p.device, copy=True).view(st[k].dtype) for k in ('exp_avg', 'exp_avg_root', 'scales')}
    first, second = (torch.empty_like(p, dtype=torch.float32) for _ in range(2))
    if 'scales' in st:
        sc = st['scales']
        for to, k, col in ((first, 'exp_avg', 0), (second, 'exp_avg_root', 1)):
            x = torch.empty_like(st[k], dtype=torch.float32)
            _memory_order(x).copy_(dequantize_moment(st[k], sc[:, col]))
            to.copy_(x)
    else:
        first.copy_(st['exp_avg'])
        second.copy_(st['exp_avg_sq'])
        if bits == 8:
            second.sqrt_()
    if bits == 32:
        return {'exp_avg': first, 'exp_avg_sq': second.square_() if 'scales' in st else second}
    out = {}
    for x, k in ((first, 'exp_avg'), (second, 'exp_avg_root')):
        codes, sc = quantize_moment(_memory_order(x), keep_positive=k == 'exp_avg_root')
        out[k] = torch.empty_like(p, dtype=torch.uint8).view(_CODE)
        _memory_order(out[k].view(torch.uint8)).copy_(codes.view(torch.uint8))
        out.setdefault('scales', torch.empty(sc.numel(), 2, dtype=torch.uint8, device=p.device).view(_SCALE))
        out['scales'].view(torch.uint8)[:, 0 if k == 'exp_avg' else 1] = sc.view(torch.uint8)
    return out
