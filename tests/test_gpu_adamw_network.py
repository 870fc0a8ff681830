"""The many-tensor optimizer step and this framework's own network: packed weights, the flat gradient buffer, copies of both."""
import copy

import pytest
import torch

pytestmark = pytest.mark.gpu

SHAPE = (1, 3, 32, 48)


@pytest.fixture(scope='module')
def optim():
    from unetk import optim
    return optim


def make_net(channels_last=False, seed=0):
    from unet import UNet
    torch.manual_seed(seed)
    net = UNet(3, 2, False).cuda().eval()
    return net.to(memory_format=torch.channels_last) if channels_last else net


def image(seed=1):
    return torch.randn(SHAPE, generator=torch.Generator().manual_seed(seed)).cuda().to(memory_format=torch.channels_last)


def forward(net, x):
    with torch.no_grad(), torch.autocast('cuda', dtype=torch.bfloat16):
        return net(x)


def fresh(net, x):
    """What a network that never saw a graph computes with these parameters."""
    other = make_net()
    other.load_state_dict(net.state_dict())
    return forward(other, x)


def fresh_gradient(net, x):
    other = make_net()
    other.load_state_dict(net.state_dict())
    return input_gradient(other, x)


def input_gradient(net, x):
    y = x.detach().clone().requires_grad_(True)
    with torch.autocast('cuda', dtype=torch.bfloat16):
        out = net(y)
    return torch.autograd.grad(out.float().square().sum(), y)[0]


def random_gradients(net, seed):
    g = torch.Generator().manual_seed(seed)
    for p in net.parameters():
        new = torch.randn(p.shape, generator=g).cuda()
        if p.grad is None:
            p.grad = torch.empty_like(p)
        p.grad.copy_(new)


@pytest.mark.parametrize('channels_last', [False, True])
def test_the_network_follows_a_replayed_step(optim, channels_last):
    """Weights that a graph writes: no eager pass may take an earlier packing of them for current, forwards or backwards."""
    net, x = make_net(channels_last), image()
    opt = optim.AdamW(net.parameters(), lr=1e-3)
    random_gradients(net, 0)
    opt.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    for k in range(3):
        before = forward(net, x)                       # fills the cache of packed weights
        input_gradient(net, x)
        random_gradients(net, k + 1)
        graph.replay()
        torch.cuda.synchronize()
        after = forward(net, x)
        assert not torch.equal(before, after)
        assert torch.equal(after, fresh(net, x)), k
        assert torch.equal(input_gradient(net, x), fresh_gradient(net, x)), k


@pytest.mark.parametrize('channels_last', [False, True])
@pytest.mark.parametrize('captured_step', [False, True])
def test_a_captured_forward_follows_the_step(optim, channels_last, captured_step):
    """A graph of the forward packs the weights it reads, whether a graph or an eager step wrote them last."""
    net, x = make_net(channels_last), image()
    opt = optim.AdamW(net.parameters(), lr=1e-3)
    random_gradients(net, 0)
    opt.step()
    forward(net, x)
    forward(net, x)
    infer, step = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(infer):                      # captured with current packings at hand
        out = forward(net, x)
    if captured_step:
        with torch.cuda.graph(step):
            opt.step()
    for k in range(3):
        random_gradients(net, k + 1)
        step.replay() if captured_step else opt.step()
        infer.replay()
        torch.cuda.synchronize()
        want = fresh(net, x)
        assert torch.equal(out, want), k
        assert torch.equal(forward(net, x), want), k


@pytest.mark.parametrize('channels_last', [False, True])
def test_a_packing_that_was_only_recorded_is_not_taken_for_done(optim, channels_last):
    net, x = make_net(channels_last), image()
    opt = optim.AdamW(net.parameters(), lr=1e-3)
    forward(net, x)
    random_gradients(net, 0)
    opt.step()                                         # the packings at hand are old now
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        forward(net, x)
    assert torch.equal(forward(net, x), fresh(net, x))


def test_a_forward_captured_before_any_other(optim):
    """No plan of the packings is there yet, and its copy to the device cannot be captured."""
    net, x = make_net(), image()
    want = fresh(net, x)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = forward(net, x)
    for _ in range(2):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)


@pytest.mark.parametrize('kind', ['adamw', 'rmsprop'])
def test_discarded_gradients_of_a_flat_buffer_are_not_applied_again(optim, kind):
    from unetk.ddp import FlatGrads
    net = make_net()
    fg = FlatGrads(net, grads_to_autograd=False)
    kw = dict(lr=1e-2, weight_decay=0.1)
    opt = optim.AdamW(fg, **kw) if kind == 'adamw' else optim.ClipRMSprop(fg, max_norm=1.0, **kw)
    for _ in range(2):
        fg.initial_grads()
        fg.flat.normal_()
        opt.step()
        opt.step()                                     # the same gradients again, as a stock optimizer would
        kept = [p.detach().clone() for p in net.parameters()]
        opt.zero_grad()
        with pytest.raises(RuntimeError, match='no gradients'):
            opt.step()
        assert all(torch.equal(p, q) for p, q in zip(net.parameters(), kept))
    if kind == 'adamw':
        assert float(opt.state[net.outc.conv.weight]['step']) == 4.0
    # gradients of zero are gradients: the decay goes on, the next backward pass is no accumulation
    fg.initial_grads()
    fg.flat.normal_()
    opt.zero_grad(set_to_none=False)
    assert not fg.flat.any() and not any(v.any() for v in fg.views.values())
    opt.step()
    assert not any(torch.equal(p, q) for p, q in zip(net.parameters(), kept) if q.any())
    opt.zero_grad(set_to_none=False)
    fg.initial_grads()
    with pytest.raises(RuntimeError, match='accumulation'):
        fg.initial_grads()


@pytest.mark.parametrize('bits', [32, 8])
def test_copies_of_a_network_and_an_optimizer_on_its_flat_gradients(optim, bits):
    from unetk.ddp import FlatGrads
    net, x = make_net(), image()
    fg = FlatGrads(net, grads_to_autograd=False)
    opt = optim.AdamW(fg, lr=1e-3, max_norm=1.0, state_bits=bits, seed=4)

    def step(n, o, seed):
        o.zero_grad()
        n._initial_grads()                             # as the network's backward pass begins
        o.fg.flat.copy_(torch.randn(o.fg.total, generator=torch.Generator().manual_seed(seed)))
        o.step()

    def same(a, b):
        assert all(torch.equal(p, q) for p, q in zip(a.parameters(), b.parameters()))

    step(net, opt, 0)
    other, twin = copy.deepcopy((net, opt))
    assert twin.fg is not fg and other._initial_grads.__self__ is twin.fg
    opt.step(), twin.step()                            # the gradients at hand, copied too
    same(net, other)
    kept, gradients = [p.detach().clone() for p in net.parameters()], fg.flat.clone()
    for k in (1, 2):                                   # the copy trains alone
        step(other, twin, k)
    twin.zero_grad()
    with torch.autocast('cuda', dtype=torch.bfloat16):
        other(x).float().square().sum().backward()
    assert bool(twin.fg.flat.any()) and torch.equal(fg.flat, gradients)
    assert all(torch.equal(p, q) for p, q in zip(net.parameters(), kept))
    assert not torch.equal(other.outc.conv.weight, net.outc.conv.weight)
    for k in (1, 2):
        step(net, opt, k)
    same(net, other)
    assert all(float(o.state[p]['step']) == 4.0 for n, o in ((net, opt), (other, twin)) for p in n.parameters())
