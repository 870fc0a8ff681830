"""The many-tensor optimizer step without a GPU: what the entry points refuse, and the 8-bit form's helpers."""
import ctypes
import os

import numpy as np
import pytest
import torch

from conftest import PKG
from oracle import adamw_np as O


@pytest.fixture(scope='module')
def nat():
    if not os.path.exists(os.path.join(PKG, 'libunetk.so')):
        import __graft_entry__
        __graft_entry__.build()
    from unetk import _native
    return _native


@pytest.fixture(scope='module')
def optim(nat):
    from unetk import optim
    return optim


def words(*values):
    return (ctypes.c_int64 * len(values))(*values)


ROW = (64, 64, 64, 64, 64, 10)                      # param, exp_avg, exp_avg_sq, scales, step, numel


def test_entry_points_refuse_before_launch(nat):
    fn, a = nat.fn, ctypes.addressof
    good, grad = words(*ROW), words(64)

    def prepare(t=good, g=grad, n=1, dtype=nat.F32, coefs=64, partials=None):
        return fn['unetk_adamw_prepare'](a(t) if t else None, a(g) if g else None, n, dtype, 1e-3, None, 0.9, 0.999, 0.0, 0, None,
                                         coefs, partials, None)

    def update(t=good, g=grad, n=1, dtype=nat.F32, coefs=64, partials=None, count=0, max_norm=1.0):
        return fn['unetk_adamw_update'](a(t) if t else None, a(g) if g else None, n, dtype, 0.9, 0.999, 1e-8, None, None, coefs, partials, count,
                        max_norm, None, None)

    assert prepare(None) == -5 and prepare(g=None) == -5 and prepare(n=0) == -5 and prepare(dtype=9) == -2
    assert prepare(coefs=None) == -5 and prepare(coefs=72) == -3 and prepare(partials=12) == -3
    assert prepare(words(*ROW[:4], 0, 10)) == -5 and prepare(words(*ROW[:4], 66, 10)) == -3            # step
    assert prepare(words(*ROW[:5], -1)) == -5 and prepare(words(*ROW[:5], 1 << 60)) == -1              # numel
    assert prepare(g=words(0)) == -5 and prepare(g=words(66)) == -3
    for scales in (0, 64):
        row = (*ROW[:3], scales, *ROW[4:])
        assert update(None) == -5 and update(g=None) == -5 and update(n=-1) == -5 and update(dtype=3) == -2
        assert update(coefs=None) == -5
        assert update(partials=64, count=0) == -5 and update(partials=None, count=4) == -5
        assert update(partials=12, count=4) == -3
        for bad in (-1.0, float('nan')):
            assert update(partials=64, count=4, max_norm=bad) == -5
        for k in range(3):
            r = list(row)
            r[k] = 0
            assert update(words(*r)) == -5
        assert update(g=words(0)) == -5
        assert update(words(*row, 66, *row[1:]), words(64, 64), 2) == -3                         # an fp32 parameter at two bytes
    assert update(words(64, 66, 64, 0, 64, 10)) == -3 and update(words(64, 64, 66, 0, 64, 10)) == -3       # fp32 moments at two bytes
    assert fn['unetk_grad_partials'](0) == -5 and 0 < fn['unetk_grad_partials'](1) <= fn['unetk_grad_partials'](1000)
    ten = words(10)
    assert fn['unetk_grad_sumsq'](a(grad), a(ten), 1, nat.F32, None, None) == -5
    assert fn['unetk_grad_sumsq'](a(grad), a(ten), 1, nat.F32, 12, None) == -3
    assert fn['unetk_grad_sumsq'](a(grad), None, 1, nat.F32, 64, None) == -5
    assert fn['unetk_grad_clip'](a(grad), a(ten), 1, nat.F32, None, 0, 1.0, None, None) == -5
    assert fn['unetk_grad_clip'](a(grad), a(ten), 1, nat.BF16, 64, 3, float('nan'), None, None) == -5


@pytest.mark.parametrize('begin,numel', [((64, 64), (10, 10)), ((64, 100), (10, 10)), ((100, 64), (10, 10)), ((64, 200, 72), (10, 3, 1)),
                                         ((4000, 64, 8000, 3996), (100, 10, 5, 2)), ((64, 4000, 64, 8000), (1, 5, 1000, 7)),
                                         ((64, 64, 64), (0, 3, 1))])
def test_gradients_that_overlap_are_refused(nat, begin, numel):
    b, n = words(*begin), words(*numel)
    assert nat.fn['unetk_grad_sumsq'](ctypes.addressof(b), ctypes.addressof(n), len(begin), nat.F32, 64, None) == -5
    if begin == (64, 100):                                                  # in 16 bits 19 elements end at 102
        n = words(19, 10)
        assert nat.fn['unetk_grad_sumsq'](ctypes.addressof(b), ctypes.addressof(n), 2, nat.BF16, 64, None) == -5


def test_overlaps_of_what_a_step_writes(nat):
    """Every pair of arrays of two records, one byte too far and one byte apart, in both forms and element sizes."""
    def overlaps(records, sizes):
        flat = words(*[w for r in records for w in r])
        es = (ctypes.c_uint8 * len(sizes))(*sizes)
        return nat.fn['unetk_adamw_overlaps'](ctypes.addressof(flat), ctypes.addressof(es), len(sizes))

    n = 300
    for es in (4, 2):
        for codes in (False, True):
            span = [n * es, n * (1 if codes else 4), n * (1 if codes else 4), 4 if codes else 0, 4]       # two blocks of scales
            def record(at):
                return [at, at + 10000, at + 20000, at + 30000 if codes else 0, at + 40000, n]
            a, b = record(1 << 20), record(1 << 24)
            assert overlaps([a, b], [es, es]) == 0 and overlaps([a], [es]) == 0
            for i in range(5):
                for j in range(5):
                    if span[i] == 0 or span[j] == 0:
                        continue
                    b2 = list(b)
                    b2[j] = a[i] + span[i]
                    assert overlaps([a, b2], [es, es]) == 0 and overlaps([b2, a], [es, es]) == 0
                    b2[j] -= 1
                    assert overlaps([a, b2], [es, es]) == 1 and overlaps([b2, a], [es, es]) == 1
                    if i < j:
                        a2 = list(a)
                        a2[j] = a[i]
                        assert overlaps([a2], [es]) == 1
            empty = [*b[:5], 0]
            assert overlaps([a, [a[0], a[1], a[2], a[3], b[4], 0]], [es, es]) == 0                       # no elements: only the count
            assert overlaps([a, [*empty[:4], a[4], 0]], [es, es]) == 1
    assert overlaps([a], []) == -5 and nat.fn['unetk_adamw_overlaps'](None, 64, 1) == -5 and nat.fn['unetk_adamw_overlaps'](64, None, 1) == -5


def test_a_subnormal_eps_with_8bit_moments_is_refused(nat, optim):
    """The reciprocal of a subnormal is infinite in the 8-bit update: 0 / eps would be NaN where a gradient was never seen."""
    row, grad, a = words(*ROW), words(64), ctypes.addressof
    for eps in (1e-40, 1e-46, 2.0 ** -126 * (1 - 2.0 ** -24)):
        assert nat.fn['unetk_adamw_update'](a(row), a(grad), 1, nat.F32, 0.9, 0.999, eps, None, None, 64, None, 0, 1.0, None, None) == -5
        with pytest.raises(ValueError, match='eps'):
            optim._usable_eps({'eps': eps}, 8)
        assert optim._usable_eps({'eps': eps}, 32) == eps
    assert optim._usable_eps({'eps': 0}, 8) == 0.0 and optim._usable_eps({'eps': 2.0 ** -126}, 8) == 2.0 ** -126


def test_no_cpu_fallback_and_bad_arguments(optim):
    p = torch.nn.Parameter(torch.zeros(4))
    with pytest.raises(RuntimeError, match='cuda'):
        optim.AdamW([p])
    p.grad = torch.ones(4)
    with pytest.raises(RuntimeError, match='cuda'):
        optim.clip_grad_norm_([p], 1.0)
    for kw in (dict(lr=-1.0), dict(eps=-1.0), dict(weight_decay=-0.1), dict(state_bits=16), dict(lr=float('nan'))):
        with pytest.raises(ValueError):
            optim.AdamW([p], **kw)
    for kw in (dict(norm_type=1.0), dict(norm_type=float('inf'))):
        with pytest.raises(ValueError):
            optim.clip_grad_norm_([p], 1.0, **kw)
    for bad in (-1.0, float('nan')):
        with pytest.raises(ValueError):
            optim.clip_grad_norm_([p], bad)
    assert float(optim.clip_grad_norm_([torch.nn.Parameter(torch.zeros(2))], 1.0)) == 0.0


def test_dense_layouts(optim):
    t = torch.zeros(3, 4, 5, 6)
    assert optim._is_dense(t) and optim._is_dense(t.to(memory_format=torch.channels_last)) and optim._is_dense(t.permute(2, 0, 3, 1))
    assert not optim._is_dense(t[:, :, :, ::2]) and not optim._is_dense(t[:, 1:]) and not optim._is_dense(torch.zeros(1).expand(4))
    assert optim._is_dense(torch.zeros(0)) and optim._is_dense(torch.zeros(()))


@pytest.mark.parametrize('n', [0, 1, 255, 256, 257, 5000])
def test_moments_to_codes_and_back(optim, n):
    """Nearest rounding: half of e4m3's step (2^-4 relative, 2^-10 of the scale below its normal range)."""
    rng = np.random.default_rng(n)
    x = (rng.standard_normal(n) * 10.0 ** rng.uniform(-12, 3, n)).astype(np.float32)
    x[: n // 3] *= 1e-30
    codes, scales = optim.quantize_moment(torch.from_numpy(x))
    assert codes.dtype == torch.float8_e4m3fn and scales.dtype == torch.float8_e8m0fnu and scales.numel() == -(-n // 256)
    k = scales.view(torch.uint8).numpy().astype(int) - 127
    assert np.array_equal(k, O.scale_exponent(x.astype(np.float64)))
    back = optim.dequantize_moment(codes, scales).numpy().astype(np.float64)
    unit = np.exp2(np.repeat(k, 256)[:n].astype(float))
    assert (np.abs(back - x) <= np.abs(x) * 2.0 ** -4 + unit * 2.0 ** -10).all()


def test_codes_of_special_values(optim):
    x = torch.zeros(512)
    x[0], x[1], x[2], x[3] = float('inf'), float('nan'), 1e-30, 2.0
    codes, scales = optim.quantize_moment(x, keep_positive=True)
    back = optim.dequantize_moment(codes, scales)
    assert torch.isnan(back[:2]).all() and back[3] == 2.0 and 0 < back[2] < 2.0 ** -15 and not back[4:].any()
    assert int(scales.view(torch.uint8)[1]) == 0
    codes, _ = optim.quantize_moment(x)
    assert float(codes[2]) == 0.0


@pytest.mark.parametrize('k', [-127, -20, 0, 100])
def test_the_oracles_rounding_is_unbiased_and_on_the_grid(k):
    """Averaged over all fractions a code is its value, to the fractions' own 2^-17 of a step; codes are e4m3's."""
    rng = np.random.default_rng(5)
    y = rng.uniform(-448, 448, 64) * 10.0 ** -rng.uniform(0, 6, 64)
    u = (np.arange(65536) + 0.5) / 65536
    for v in y:
        q = O.round_code(np.full(65536, v), u, False)
        assert np.array_equal(q.astype(np.float32), torch.from_numpy(q).float().to(torch.float8_e4m3fn).float().numpy())
        ulp = np.exp2(max(np.frexp(abs(v))[1] - 4, -9))
        assert abs(q.mean() - v) <= ulp * 2.0 ** -16
    x = np.ldexp(y[:1], k)
    assert O.scale_exponent(np.array([np.ldexp(448.0, k)]))[0] == k and O.scale_exponent(np.array([np.ldexp(448.5, k)]))[0] == k + 1
    assert O.scale_exponent(x * 0)[0] == -127


def test_the_oracles_step_is_torchs():
    g = torch.Generator().manual_seed(3)
    p = torch.nn.Parameter(torch.randn(300, generator=g, dtype=torch.float64))
    opt = torch.optim.AdamW([p], lr=1e-2, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.1)
    v = dict(p=p.detach().numpy().copy(), m=np.zeros(300), v=np.zeros(300))
    for t in range(1, 6):
        p.grad = torch.randn(300, generator=g, dtype=torch.float64)
        v = O.step(v['p'], p.grad.numpy(), v['m'], v['v'], t, 1e-2, 0.9, 0.99, 1e-8, 0.1)
        opt.step()
        assert np.allclose(v['p'], p.detach().numpy(), rtol=1e-12, atol=1e-14)
    st = opt.state[p]
    assert np.allclose(st['exp_avg'], v['m'], rtol=1e-12) and np.allclose(st['exp_avg_sq'], v['v'], rtol=1e-12)


@pytest.mark.parametrize('flat', [False, True])
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_what_shrinks_where_it_lies_ends_a_plan(optim, flat, dtype):
    """A parameter or a gradient that is smaller at the same address (pruned and moved back, or of another type): the kernels would
    write past its end with the table of the step before."""
    from types import SimpleNamespace
    params = [torch.nn.Parameter(torch.zeros(n, dtype=dtype)) for n in (40, 30)]
    opt = SimpleNamespace(fg=None, _apart=None, param_groups=[{'params': params}], state={})
    for p in params:
        p.grad = torch.zeros_like(p)
        opt.state[p] = {'step': torch.zeros(()), 'exp_avg': torch.zeros(p.shape), 'exp_avg_sq': torch.zeros(p.shape)}
    if flat:
        opt.fg = SimpleNamespace(offsets={id(params[0]): 0, id(params[1]): 40}, flat=torch.zeros(72, dtype=dtype))
    plan = optim._Plan(opt, {(0, dtype): [(p, opt.state[p], p.grad) for p in params]}, [])
    assert plan.pointers(opt) is not None
    p, whole, half = params[1], params[1].data, torch.bfloat16 if dtype == torch.float32 else torch.float16
    p.data = whole[:29]
    assert plan.pointers(opt) is None
    if dtype == torch.float32:
        p.data = whole.view(half)[:30]
        assert plan.pointers(opt) is None
    p.data = whole
    assert plan.pointers(opt) is not None
    if not flat:
        grad = p.grad.data
        p.grad.data = grad[:29]
        assert plan.pointers(opt) is None
        p.grad.data = grad.view(half)[:30]
        assert plan.pointers(opt) is None
        p.grad.data = grad
        assert plan.pointers(opt) is not None
        p.grad = None
        assert plan.pointers(opt) is None


def test_a_pass_over_the_network_is_its_threads_own(nat):
    """Two passes that overlap in time, and end in the order they began, leave nothing behind."""
    import threading
    from unetk import blocks
    inside, leave, seen = threading.Event(), threading.Event(), []

    def other():
        with blocks.planned(frozenset({'b'})):
            inside.set()
            leave.wait(10)
            seen.append(blocks._PASS.packed)
        seen.append(blocks._PASS.packed)

    t = threading.Thread(target=other)
    with blocks.planned(frozenset({'a'})):
        t.start()
        inside.wait(10)
        assert blocks._PASS.packed == {'a'}
        with pytest.raises(ZeroDivisionError):
            with blocks.planned(frozenset({'c'})):
                1 / 0
        assert blocks._PASS.packed == {'a'}
    leave.set()
    t.join()
    assert seen == [{'b'}, frozenset()] and blocks._PASS.packed == frozenset()
