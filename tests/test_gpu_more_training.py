"""The loss of a linear layer, distillation and the group norm together, in networks, threads and graphs, under autocast, and beyond 2^31 values."""
import math

import pytest
import torch as ch
from test_gpu_training_threads import side_by_side

pytestmark = pytest.mark.gpu


class Network(ch.nn.Module):
    """A convolutional stem with group norms, and two heads: one whose loss makes its logits itself, one that is taught."""

    def __init__(self, classes, dtype, plain=False):
        from ffcv_b200.training import GroupNormAct, LinearCrossEntropy
        super().__init__()
        ch.manual_seed(0)
        norm = (lambda c: ch.nn.Sequential(ch.nn.GroupNorm(8, c), ch.nn.SiLU())) if plain else (lambda c: GroupNormAct(8, c, 'silu'))
        self.first, self.second = ch.nn.Conv2d(3, 32, 3, 2, 1), ch.nn.Conv2d(32, 64, 3, 2, 1)
        self.norms = ch.nn.ModuleList([norm(32), norm(64)])
        self.head = ch.nn.Linear(64, classes) if plain else LinearCrossEntropy(64, classes, label_smoothing=0.1)
        self.to(device='cuda', dtype=dtype, memory_format=ch.channels_last)
        self.plain = plain

    def forward(self, images, labels, best, where):
        from ffcv_b200.training import distillation
        x = self.norms[1](self.second(self.norms[0](self.first(images)))).mean((2, 3))
        if not self.plain:
            return self.head(x, labels) + distillation(self.head.logits(x), best, where, temperature=2.0)
        z = self.head(x)
        q, log_p = ch.softmax(best.to(z.dtype) / 2, 1), ch.log_softmax(z / 2, 1)
        taught = 4 * (q * (ch.log(q) - log_p.gather(1, where.long()))).sum(1).mean()
        return ch.nn.functional.cross_entropy(z, labels, label_smoothing=0.1) + taught


def batch(n, classes, dtype, side=32):
    gen = ch.Generator('cuda').manual_seed(3)
    images = ch.randn(n, side, side, 3, generator=gen, device='cuda').to(dtype).permute(0, 3, 1, 2)
    best, where = (ch.randn(n, classes, generator=gen, device='cuda') * 3).topk(8, 1)
    return images, ch.randint(classes, (n,), generator=gen, device='cuda'), best, where.int()


def test_a_network_and_its_gradients():
    """Against the same network of plain operations in 64 bits.  Values of 16 bits on the way are off by 2^-9 each (bfloat16); through a handful of layers
    gradients agree to some percent of their norm."""
    got, want = Network(200, ch.bfloat16), Network(200, ch.float64, plain=True)
    names = {'norms.0.0.': 'norms.0.', 'norms.1.0.': 'norms.1.'}
    state = {}
    for name in want.state_dict():
        mine = name
        for a, b in names.items():
            mine = mine.replace(a, b)
        state[name] = got.state_dict()[mine].double()
    want.load_state_dict(state)
    images, labels, best, where = batch(64, 200, ch.bfloat16)
    loss = got(images, labels, best, where)
    loss.backward()
    exact = want(images.double(), labels, best.double(), where)
    exact.backward()
    assert abs(float(loss) - float(exact)) < 0.02 * float(exact)
    grads = dict(got.named_parameters())
    for name, p in want.named_parameters():
        mine = name
        for a, b in names.items():
            mine = mine.replace(a, b)
        g = grads[mine].grad.double()
        assert (g - p.grad).norm() < 0.06 * p.grad.norm() + 1e-4, name


def test_a_step_in_a_graph():
    """Forward and backward of all of them captured once, replayed on other data."""
    net = Network(300, ch.bfloat16)
    data = batch(64, 300, ch.bfloat16)
    side = ch.cuda.Stream()
    side.wait_stream(ch.cuda.current_stream())
    with ch.cuda.stream(side):
        for _ in range(2):
            net.zero_grad(set_to_none=True)
            net(*data).backward()
    ch.cuda.current_stream().wait_stream(side)
    net.zero_grad(set_to_none=True)
    graph = ch.cuda.CUDAGraph()
    with ch.cuda.graph(graph):
        loss = net(*data)
        loss.backward()
    kept = [p.grad for p in net.parameters()]
    data[0].copy_(ch.randn_like(data[0]))
    data[1].copy_(ch.randint(300, (64,), device='cuda'))
    graph.replay()
    ch.cuda.synchronize()
    got = [loss.clone()] + [g.clone() for g in kept]
    net.zero_grad(set_to_none=True)
    again = net(*data)
    again.backward()
    for a, b in zip(got, [again] + [p.grad for p in net.parameters()]):
        assert ch.allclose(a.float(), b.float(), rtol=0.05, atol=0.02 * float(b.float().abs().max()))  # (convolutions may take another way)


def test_autocast():
    from ffcv_b200.training import LinearCrossEntropy
    layer = LinearCrossEntropy(64, 50, device='cuda')
    x, y = ch.randn(30, 64, device='cuda', requires_grad=True), ch.randint(50, (30,), device='cuda')
    with pytest.raises(TypeError, match='float16 or bfloat16'):
        layer(x, y)
    with ch.autocast('cuda', dtype=ch.bfloat16):
        loss = layer(x, y)
    loss.backward()
    assert layer.weight.grad.dtype == ch.float32 and x.grad.dtype == ch.float32
    z = x.detach().bfloat16().double() @ layer.weight.detach().bfloat16().double().t() + layer.bias.detach().bfloat16().double()
    assert abs(float(loss) - float(ch.nn.functional.cross_entropy(z, y))) < 1e-5


def test_refusals():
    from ffcv_b200.training import distillation, group_norm_act, group_norm_act_backward, linear_cross_entropy
    x, w, y = (ch.randn(*s, device='cuda', dtype=ch.bfloat16) for s in ((8, 16), (20, 16), (8,)))
    labels = ch.zeros(8, dtype=ch.long, device='cuda')
    for bad, error in ((dict(), ValueError), (dict(labels=labels, mixed=ch.zeros(8, 3, device='cuda')), ValueError), (dict(labels=labels[:4]), ValueError),
                       (dict(labels=labels.float()), TypeError), (dict(labels=labels.cpu()), ValueError), (dict(mixed=ch.zeros(8, 2, device='cuda')), ValueError),
                       (dict(labels=labels, label_smoothing=1.5), ValueError), (dict(labels=labels, reduction='median'), ValueError),
                       (dict(mixed=ch.zeros(8, 3, device='cuda'), ignore_index=0), ValueError), (dict(labels=labels, bias=y), ValueError),
                       (dict(labels=labels, bias=ch.zeros(20, device='cuda')), TypeError)):
        with pytest.raises(error):
            linear_cross_entropy(x, w, **bad)
    for hidden, weight in ((x.float(), w.float()), (x, w.half()), (x.double(), w)):
        with pytest.raises(TypeError):
            linear_cross_entropy(hidden, weight, labels)
    for hidden, weight in ((x[None], w), (x, w[:, :8]), (x, w[:0]), (x[:, :0], w[:, :0])):
        with pytest.raises(ValueError):
            linear_cross_entropy(hidden, weight, labels)
    z, t, c = ch.randn(8, 30, device='cuda'), ch.randn(8, 4, device='cuda'), ch.zeros(8, 4, dtype=ch.int32, device='cuda')
    for args, how, error in (((z, t, c.float()), {}, TypeError), ((z, t, c[:, :3]), {}, ValueError), ((z, t[:4], c[:4]), {}, ValueError), ((z, t[:, :0], c[:, :0]), {}, ValueError),
                             ((z, t.double(), c), {}, TypeError), ((z, t, c), dict(temperature=0.0), ValueError), ((z, t, c), dict(temperature=math.nan), ValueError),
                             ((z, t, c), dict(hard_weight=0.5), ValueError), ((z, t, c, labels), dict(hard_weight=1.5), ValueError),
                             ((z, t, c, labels), dict(mixed=ch.zeros(8, 3, device='cuda')), ValueError), ((z, t, c), dict(ignore_index=1), ValueError),
                             ((z, t.clone().requires_grad_(), c), {}, ValueError), ((z, ch.randn(8, 1025, device='cuda'), ch.zeros(8, 1025, dtype=ch.int32, device='cuda')), {}, ValueError),
                             ((z[:, :0], t.detach(), c), {}, ValueError), ((z, t.detach(), c.cpu()), {}, ValueError)):
        with pytest.raises(error):
            distillation(*args, **how)
    image = ch.randn(2, 12, 5, 5, device='cuda')
    for args, how, error in (((image, 5), {}, ValueError), ((image, 0), {}, ValueError), ((image, 2.0), {}, ValueError), ((image[0, 0, 0], 1), {}, ValueError),
                             ((image, 2, image[0, 0, 0]), {}, ValueError), ((image, 2, ch.ones(12, device='cuda'), ch.ones(12, device='cuda').half()), {}, TypeError),
                             ((image, 2), dict(activation='tanh'), ValueError), ((image, 2), dict(eps=-1.0), ValueError), ((image.double(), 2), {}, TypeError),
                             ((image, 2, ch.ones(12)), {}, TypeError)):
        with pytest.raises(error):
            group_norm_act(*args, **how)
    for dy, stats in ((image.half(), ch.zeros(2, 2, 2, device='cuda')), (image[:1], ch.zeros(2, 2, 2, device='cuda')), (image, ch.zeros(2, 2, device='cuda'))):
        with pytest.raises(ValueError):
            group_norm_act_backward(dy, image, stats, 2)


def test_threads():
    """Calls of other sizes at once: none lowers what another one's kernel may have."""
    from ffcv_b200.training import distillation_with_grad, group_norm_act_backward, group_norm_act_forward, linear_cross_entropy_with_grad
    calls = []
    for classes, width in ((500, 64), (4000, 136)):
        x, w, y = ch.randn(300, width, device='cuda').bfloat16(), ch.randn(classes, width, device='cuda').bfloat16(), ch.randint(classes, (300,), device='cuda')
        calls.append(lambda x=x, w=w, y=y: linear_cross_entropy_with_grad(x, w, y)[1:3])
    for classes, kept in ((18000, 20), (12000, 600)):
        z, t, c = ch.randn(100, classes, device='cuda'), ch.randn(100, kept, device='cuda'), ch.randint(classes, (100, kept), device='cuda')
        calls.append(lambda z=z, t=t, c=c: distillation_with_grad(z, t, c, temperature=2.0))
    for sides in ((20, 20), (60, 60)):
        x, dy = (ch.randn(2, *sides, 64, device='cuda').permute(0, 3, 1, 2) for _ in range(2))
        calls.append(lambda x=x, dy=dy: group_norm_act_backward(dy, x, group_norm_act_forward(x, 4, activation='silu')[1], 4, activation='silu').values())
    want = [[v.clone() for v in call()] for call in calls]
    assert not side_by_side(calls, 300)
    assert all(ch.equal(a, b) for call, first in zip(calls, want) for a, b in zip(call(), first))


@pytest.fixture
def room():
    if ch.cuda.get_device_properties(0).total_memory < 100 << 30:
        pytest.skip('needs 100 GB')
    yield
    ch.cuda.empty_cache()


def test_head_beyond_32_bits(room):
    """More than 2^31 logits, and rows of weights of which the last ones begin behind 2^31 values: the last samples' losses and gradients are those of a small call
    with the same classes; the last classes' gradients those by the formula."""
    from ffcv_b200.training import linear_cross_entropy_with_grad
    rows, classes, width = 70_000, 40_000, 64
    x, w, y = ch.randn(rows, width, device='cuda').bfloat16(), (ch.randn(classes, width, device='cuda') * 0.3).bfloat16(), ch.randint(classes, (rows,), device='cuda')
    loss, dx, dw, _ = linear_cross_entropy_with_grad(x, w, y, reduction='none')
    small, small_dx, _, _ = linear_cross_entropy_with_grad(x[-300:].clone(), w, y[-300:].clone(), reduction='none')
    assert rows * classes > 1 << 31
    assert ch.allclose(loss[-300:], small, rtol=1e-5) and ch.allclose(dx[-300:].float(), small_dx.float(), rtol=2 ** -7, atol=2e-3)
    some = ch.cat([ch.arange(5), ch.arange(classes - 50, classes)]).cuda()
    want, size = (ch.zeros(len(some), width, dtype=ch.float64, device='cuda') for _ in range(2))
    for part in range(0, rows, 2000):
        xs = x[part:part + 2000].double()
        z = xs @ w.double().t()
        g = ch.exp(z[:, some] - ch.logsumexp(z, 1, keepdim=True)) - (y[part:part + 2000, None] == some).double()
        want += g.t() @ xs
        size += g.abs().t() @ xs.abs()
    assert ((dw[some].double() - want).abs() <= 2 ** -8 * want.abs() + 2 ** -8 * size + 1e-3).all()
    wide = ch.randn(40_000, 60_000, device='cuda', dtype=ch.bfloat16)
    loss, dx, dw, _ = linear_cross_entropy_with_grad(ch.zeros(3, 60_000, device='cuda', dtype=ch.bfloat16), wide, ch.tensor([0, 39_999, 5], device='cuda'), reduction='sum')
    assert wide.numel() > 1 << 31 and abs(float(loss) - 3 * math.log(40_000)) < 1e-3
    want = wide.float().mean(0) * 3 - wide[[0, 39_999, 5]].float().sum(0)
    assert ch.allclose(dx.float().sum(0), want, rtol=0.02, atol=0.05)


def test_distillation_beyond_32_bits(room):
    from ffcv_b200.training import distillation_with_grad
    rows, classes, kept = 66_000, 33_001, 40
    z = ch.zeros((rows, classes), dtype=ch.bfloat16, device='cuda')
    z[-5:] = ch.randn((5, classes), device='cuda') * 3
    t, c = ch.randn(rows, kept, device='cuda'), ch.randint(classes, (rows, kept), device='cuda')
    loss, grad = distillation_with_grad(z, t, c, temperature=2.0, reduction='none')
    # (80 rows: with fewer a row is shared by more CTAs, or begins elsewhere between boundaries of 16 bytes)
    small, small_grad = distillation_with_grad(z[-80:].clone(), t[-80:], c[-80:], temperature=2.0, reduction='none')
    assert z.numel() > 1 << 31 and ch.equal(grad[-5:], small_grad[-5:]) and ch.allclose(loss[-5:], small[-5:], rtol=1e-6)


def test_group_norm_beyond_32_bits(room):
    """One sample of more than 2^31 values, and many samples."""
    from ffcv_b200.training import group_norm_act_backward, group_norm_act_forward
    for shape, groups in (((1, 5800, 5800, 64), 2), ((70_000, 2, 2, 8), 4)):
        x = ch.randn(shape, device='cuda', dtype=ch.float16).permute(0, 3, 1, 2)
        x[-1, -1, -1, -1] = 100.0
        dy = ch.randn(shape, device='cuda', dtype=ch.float16).permute(0, 3, 1, 2)
        w = ch.ones(shape[3], device='cuda', dtype=ch.float16)
        y, stats = group_norm_act_forward(x, groups, weight=w, activation='silu')
        grads = group_norm_act_backward(dy, x, stats, groups, weight=w, activation='silu')
        some = (slice(-1, None), slice(-shape[3] // groups, None), slice(-2, None), slice(-2, None))
        flat = x[-1].movedim(0, -1).reshape(-1, groups, shape[3] // groups)[:, -1]
        mean, var = flat.double().mean(), flat.double().var(correction=0)
        assert abs(float(stats[-1, -1, 0]) - float(mean)) < 1e-5 and abs(float(stats[-1, -1, 1]) * math.sqrt(float(var) + 1e-5) - 1) < 1e-5
        hat = (x[some].double() - mean) / (var + 1e-5).sqrt()
        assert ch.allclose(y[some].double(), ch.nn.functional.silu(hat), rtol=2e-3, atol=1e-4)
        flat_hat = (flat.float() - mean.float()) * stats[-1, -1, 1]
        gate = ch.sigmoid(flat_hat)
        da = dy[-1].movedim(0, -1).reshape(-1, groups, shape[3] // groups)[:, -1].float() * gate * (1 + flat_hat * (1 - gate))
        less, less_hat = da.double().mean(), (da * flat_hat).double().mean()
        gate = ch.sigmoid(hat)
        want = (dy[some].double() * gate * (1 + hat * (1 - gate)) - less - hat * less_hat) / (var + 1e-5).sqrt()
        assert ch.allclose(grads['x'][some].double(), want, rtol=2e-3, atol=1e-3)
