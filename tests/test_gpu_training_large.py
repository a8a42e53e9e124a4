"""The training operators beyond 2^31 and 2^32 values, and in captured graphs.  Rows (tokens, blocks) do not depend on one another, so the
last ones of a large call have to be those of a small call, bit for bit."""
import numpy as np
import pytest
import torch as ch

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def room():
    if ch.cuda.get_device_properties(0).total_memory < 100 << 30:
        pytest.skip('needs 100 GB')
    yield
    ch.cuda.empty_cache()


def test_loss():
    from ffcv_b200.training import cross_entropy_with_grad
    rows, classes = 66_000, 33_001
    x = ch.zeros((rows, classes), dtype=ch.bfloat16, device='cuda')
    x[-5:] = ch.randn((5, classes), device='cuda') * 3
    y = ch.randint(classes, (rows,), device='cuda')
    loss, grad = cross_entropy_with_grad(x, y, reduction='none')
    # (of 80 rows: with fewer a row is shared by more CTAs, and begins elsewhere between boundaries of 16 bytes unless they are a multiple of
    # eight; either decides the order of its sums)
    small, small_grad = cross_entropy_with_grad(x[-80:].clone(), y[-80:], reduction='none')
    assert x.numel() > 1 << 31 and ch.equal(loss[-5:], small[-5:]) and ch.equal(grad[-5:], small_grad[-5:])


def test_norms():
    from ffcv_b200.training import norm_residual_backward, norm_residual_forward
    rows, width = 2_100_000, 1032
    x, h, dy, dz = (ch.zeros((rows, width), dtype=ch.bfloat16, device='cuda') for _ in range(4))
    for t in (x, h, dy, dz):
        t[-6:] = ch.randn((6, width), device='cuda')
    how = dict(weight=1 + 0.2 * ch.randn(width, device='cuda'), bias=ch.randn(width, device='cuda'), scale=ch.randn(width, device='cuda'))
    y, z, stats = norm_residual_forward(x, h, **how)
    grads = norm_residual_backward(dy, dz, x, h, stats, **how)
    cut = [t[-6:].clone() for t in (x, h, dy, dz)]
    sy, sz, small = norm_residual_forward(cut[0], cut[1], **how)
    want = norm_residual_backward(cut[2], cut[3], cut[0], cut[1], small, **how)
    assert x.numel() > 1 << 31 and ch.equal(y[-6:], sy) and ch.equal(z[-6:], sz)
    assert ch.equal(grads['x'][-6:], want['x']) and ch.equal(grads['h'][-6:], want['h'])
    # the other rows have gradients of 0: the sums are the same but for their order
    assert ch.allclose(grads['weight'], want['weight'], rtol=1e-5, atol=1e-5) and ch.allclose(grads['scale'], want['scale'], rtol=1e-5, atol=1e-5)


def test_rotary():
    from ffcv_b200.training import RotaryPositions
    tokens = 6_000_000
    rotary = RotaryPositions(128, base=1e6)
    q, k = (ch.zeros((1, tokens, n, 128), dtype=ch.float16, device='cuda') for n in (3, 1))
    q[:, -9:], k[:, -9:] = ch.randn((1, 9, 3, 128), device='cuda'), ch.randn((1, 9, 1, 128), device='cuda')
    a, b = rotary.rotate(q, k)
    where = ch.arange(tokens - 9, tokens, device='cuda')
    c, d = rotary.rotate(q[:, -9:].clone(), k[:, -9:].clone(), where)
    assert q.numel() > 1 << 31 and ch.equal(a[:, -9:], c) and ch.equal(b[:, -9:], d)


@pytest.mark.parametrize('bits', [32, 8])
def test_adamw(bits):
    """One tensor; with 8 bits the noise of places beyond 2^32 is that of the upper half of the place too."""
    from ffcv_b200.training import AdamW
    n = (1 << 32) + 700 if bits == 8 else (1 << 31) + 700
    last = 700
    p = ch.nn.Parameter(ch.zeros(n, device='cuda'))
    p.data[-last:] = ch.randn(last, device='cuda')
    p.grad = ch.zeros(n, device='cuda')
    p.grad[-last:] = ch.randn(last, device='cuda')
    small = ch.nn.Parameter(p.data[-last:].clone())
    small.grad = p.grad[-last:].clone()
    a, b = AdamW([p], lr=0.1, state_bits=bits, seed=3), AdamW([small], lr=0.1, state_bits=bits, seed=3)
    a.step()
    b.step()
    assert ch.equal(p.data[-last:], small.data) and not p.data[:n - last].any()
    if bits == 32:
        assert ch.equal(a.exp_avg[n - last:n], b.exp_avg[:last]) and ch.equal(a.exp_avg_sq[n - last:n], b.exp_avg_sq[:last])
        return
    scales = a.scales[-3:].cpu()
    assert ch.equal(scales, b.scales.cpu())  # (the same blocks)
    g = np.zeros(768, np.float32)
    g[:last] = small.grad.cpu().numpy()

    def mix(x):
        x = (x * 0xE4C6EF2B) & 0xFFFFFFFF
        x ^= x >> 15
        x = (x * 0x87EA99B3) & 0xFFFFFFFF
        return x ^ (x >> 16)

    key = mix(mix(4) ^ 1)
    m = g * np.float32(1 - 0.9)
    for i in (0, 1, 255, 256, 699):
        place = n - last + i
        noise = mix(((place & 0xFFFFFFFF) + key + (place >> 32) * 0x9E3779B9) & 0xFFFFFFFF)
        down = np.float32(1 / float(scales[i // 256, 0]))
        bits_of = np.float32(abs(m[i]) * down * np.float32(2.0 ** -120)).view(np.int32)
        code = (int(bits_of) + ((noise & 0xFFFF) << 4)) >> 20 | (128 if m[i] < 0 else 0)
        assert int(a.exp_avg.view(ch.uint8)[place]) == code


def test_captured_graphs():
    """Calls that have been captured give, replayed on new values, what the calls give."""
    from ffcv_b200.training import RotaryPositions, cross_entropy_with_grad, norm_residual_backward, norm_residual_forward
    gen = ch.Generator('cuda').manual_seed(0)
    rotary = RotaryPositions(64)
    x, h, dy, dz = (ch.empty(4, 50, 192, device='cuda', dtype=ch.bfloat16) for _ in range(4))
    gate, w = ch.empty(4, 1, 192, device='cuda', dtype=ch.bfloat16), ch.ones(192, device='cuda')
    q, k, logits = ch.empty(2, 30, 3, 64, device='cuda'), ch.empty(2, 30, 1, 64, device='cuda'), ch.empty(64, 5000, device='cuda')
    labels, where = ch.randint(5000, (64,), generator=gen, device='cuda'), ch.arange(30, device='cuda')

    def calls():
        y, z, stats = norm_residual_forward(x, h, weight=w, gate=gate, post_norm='rms', post_weight=w)
        grads = norm_residual_backward(dy, dz, x, h, stats, weight=w, gate=gate, post_norm='rms', post_weight=w)
        return [y, z, *grads.values(), *rotary.rotate(q, k, where), *cross_entropy_with_grad(logits, labels, ignore_index=7)]

    def fill():
        for t in (x, h, dy, dz, gate, q, k, logits):
            t.copy_(ch.randn(t.shape, generator=gen, device='cuda'))

    fill()
    side = ch.cuda.Stream()
    side.wait_stream(ch.cuda.current_stream())
    with ch.cuda.stream(side):
        calls()
    ch.cuda.current_stream().wait_stream(side)
    graph = ch.cuda.CUDAGraph()
    with ch.cuda.graph(graph):
        out = calls()
    for _ in range(3):
        fill()
        graph.replay()
        assert all(ch.equal(a, b) for a, b in zip(out, calls()))
