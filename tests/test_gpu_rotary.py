"""Rotary positions against their definition in 64 bits (tests/_kv_ref.py), forward and backward."""
import pytest
import torch

import torch_mlu_amd as tm
from tests import _kv_ref as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, HF, FP = torch.bfloat16, torch.float16, torch.float32


def _x(shape, dtype, seed):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


def _close(got, want, tol, dtype):
    bad = ~((got.double().cpu() - want).abs() <= tol + want.abs() * torch.finfo(dtype).eps / 2 * (1 + 2.0 ** -10))
    assert not bad.any(), (float((got.double().cpu() - want).abs().max()), bad.nonzero()[:3].tolist())


def _positions(A, shape, far, seed, dtype=torch.int32):
    return torch.randint(-5, far, (A,) + shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


@pytest.mark.parametrize("dtype", [BF, HF, FP])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("D,pairs", [(128, (64,)), (128, (16, 24, 24)), (64, (8, 0, 24)), (80, (13, 27)), (256, (100, 28)), (6, (1, 2)), (96, (16, 16)), (128, (32,)),
                                     (33, (5, 9))])
def test_forward(dtype, interleaved, D, pairs):
    """All pairs of a head or a part of it (the rest is copied), sizes that 16-byte pieces take and others."""
    B, S, Hq, Hk = 2, 5, 3, 2
    freq, axes = tm.rotary_frequencies(pairs)
    q, k, pos = _x((B, Hq, S, D), dtype, 1), _x((B, Hk, S, D), dtype, 2), _positions(len(pairs), (B, S), 5000, 3)
    gq, gk = tm.rotary(q.to(DEV), k.to(DEV), pos.to(DEV), freq.to(DEV), axes.to(DEV), interleaved=interleaved)
    for x, y in ((q, gq), (k, gk)):
        want, tol = ref.rotary(x.double(), pos, freq, axes, interleaved)
        assert y.shape == x.shape and y.dtype == dtype
        _close(y, want, tol, dtype)
    n = 2 * sum(pairs)
    assert torch.equal(gq[..., n:].cpu(), q[..., n:])


@pytest.mark.parametrize("T,Hq,Hk", [(1, 1, 1), (1, 32, 8), (17, 7, 1), (300, 16, 4), (5000, 2, 1)])
def test_packed(T, Hq, Hk):
    freq, axes = tm.rotary_frequencies((32,), theta=500000.0)
    q, k, pos = _x((T, Hq, 64), BF, 4), _x((T, Hk, 64), BF, 5), _positions(1, (T,), 1 << 20, 6)
    gq, gk = tm.rotary(q.to(DEV), k.to(DEV), pos.to(DEV), freq.to(DEV), axes.to(DEV))
    for x, y in ((q, gq), (k, gk)):
        _close(y, *ref.rotary(x.double(), pos, freq, axes, False), BF)


@pytest.mark.parametrize("far,dtype", [(1 << 20, torch.int32), (1 << 30, torch.int32), (1 << 40, torch.int64)])
def test_far_positions(far, dtype):
    """Angles keep their accuracy far into a prompt: their 64-bit product has 2^-53 of the turns (here up to 2^38) left."""
    freq, axes = tm.rotary_frequencies((32,))
    x = _x((40, 2, 64), FP, 7)
    pos = (far - 1 - torch.arange(40)).to(dtype)[None]
    y, _ = tm.rotary(x.to(DEV), None, pos.to(DEV), freq.to(DEV), axes.to(DEV))
    want, tol = ref.rotary(x.double(), pos, freq, axes, False)
    _close(y, want, tol + far * 2.0 ** -51 * 2 * x.abs().max(), FP)


def test_positions_of_either_type_shared_by_the_batch_and_strided():
    freq, axes = tm.rotary_frequencies((8, 24))
    q = _x((3, 2, 9, 64), BF, 8).to(DEV)
    pos = _positions(2, (9,), 100, 9).to(DEV)
    want, _ = tm.rotary(q, None, pos[:, None].expand(2, 3, 9).contiguous(), freq.to(DEV), axes.to(DEV))
    for p in (pos, pos.long(), pos[:, None].expand(2, 3, 9), pos.t().contiguous().t(), torch.stack([pos, pos * 0], -1)[..., 0]):
        assert torch.equal(tm.rotary(q, None, p, freq.to(DEV), axes.to(DEV))[0], want)
    a, _ = tm.rotary(q, None, pos, freq.float().to(DEV), axes.to(DEV))
    _close(a, *ref.rotary(q.double().cpu(), pos.cpu()[:, None].expand(2, 3, 9), freq.float().double(), axes, False), BF)
    # an axis that is not there counts as the nearest
    assert torch.equal(tm.rotary(q, None, pos, freq.to(DEV), (axes * 9 - 4).to(DEV))[0], want)


def test_strided_inputs():
    freq, axes = (t.to(DEV) for t in tm.rotary_frequencies((32,)))
    qkv = _x((2, 7, 10, 64), BF, 10).to(DEV)
    pos = _positions(1, (2, 7), 1000, 11).to(DEV)
    q, k = qkv[:, :, :6].transpose(1, 2), qkv[:, :, 6:8].transpose(1, 2)
    want = tm.rotary(q.contiguous(), k.contiguous(), pos, freq, axes)
    got = tm.rotary(q, k, pos, freq, axes)
    odd = torch.zeros(2, 6, 7, 65, dtype=BF, device=DEV)
    odd[..., :64] = q
    last = q.transpose(2, 3).contiguous().transpose(2, 3)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert torch.equal(tm.rotary(odd[..., :64], None, pos, freq, axes)[0], want[0])
    assert torch.equal(tm.rotary(odd[..., 1:], None, pos, freq, axes)[0], tm.rotary(odd[..., 1:].contiguous(), None, pos, freq, axes)[0])
    assert torch.equal(tm.rotary(last, None, pos, freq, axes)[0], want[0])
    one = q[:, :1, :1].expand(2, 6, 7, 64)  # heads and rows that are the same memory
    assert torch.equal(tm.rotary(one, None, pos, freq, axes)[0], tm.rotary(one.contiguous(), None, pos, freq, axes)[0])


@pytest.mark.parametrize("dtype", [BF, HF, FP])
@pytest.mark.parametrize("interleaved", [False, True])
def test_backward(dtype, interleaved):
    B, S, D = 2, 6, 64
    freq, axes = tm.rotary_frequencies((4, 8, 12))
    pos = _positions(3, (B, S), 3000, 12)
    q, k = (_x((B, h, S, D), dtype, 13 + h).to(DEV).requires_grad_() for h in (4, 2))
    gq, gk = _x((B, 4, S, D), dtype, 16), _x((B, S, 2, D), dtype, 17).transpose(1, 2)
    y = tm.rotary(q, k, pos.to(DEV), freq.to(DEV), axes.to(DEV), interleaved=interleaved)
    dq, dk = torch.autograd.grad(y, (q, k), (gq.to(DEV), gk.to(DEV)))
    for g, d in ((gq, dq), (gk, dk)):
        _close(d, *ref.rotary(g.double(), pos, freq, axes, interleaved, inverse=True), dtype)


def test_backward_against_differences():
    """Along a random direction, in fp32: the map is linear, so a difference over any step is its slope but for rounding."""
    freq, axes = (t.to(DEV) for t in tm.rotary_frequencies((6, 10)))
    pos = _positions(2, (1, 9), 500, 18).to(DEV)
    x, g, d = (_x((1, 3, 9, 40), FP, s).to(DEV) for s in (19, 20, 21))
    x.requires_grad_()
    f = lambda z: (tm.rotary(z, None, pos, freq, axes)[0].double() * g.double()).sum()  # noqa: E731
    dx, = torch.autograd.grad(tm.rotary(x, None, pos, freq, axes)[0], x, g)
    with torch.no_grad():
        slope = (f(x + d) - f(x - d)) / 2
    # each element of the four turned tensors is off by 2^-21 (|a| + |b|) and 2^-24 of itself: below 2^-20 of the sizes' products
    bound = 2.0 ** -20 * 2 * float((g.abs().double() * (x.detach().abs() + d.abs()).double().sum(-1, keepdim=True)).sum())
    assert abs(float(slope - (dx.double() * d.double()).sum())) <= bound


def test_backward_of_parts():
    """One input's gradient alone, a key that takes none, expanded inputs and gradients, a second derivative."""
    freq, axes = (t.to(DEV) for t in tm.rotary_frequencies((16,)))
    pos = _positions(1, (2, 5), 500, 22).to(DEV)
    q, k = _x((2, 3, 5, 32), FP, 23).to(DEV), _x((2, 1, 5, 32), FP, 24).to(DEV)
    inv = lambda g: torch.ops.torch_mlu_amd.rotary(g.contiguous(), None, pos, freq, axes, False, True)[0]  # noqa: E731
    qg = q.clone().requires_grad_()
    a, b = tm.rotary(qg, k, pos, freq, axes)
    assert a.requires_grad and not b.requires_grad
    assert torch.equal(torch.autograd.grad(a.sum(), qg)[0], inv(torch.ones_like(q)))  # an expanded gradient
    kg = k.clone().requires_grad_()
    a, b = tm.rotary(q, kg, pos, freq, axes)
    assert b.requires_grad and not a.requires_grad
    assert torch.equal(torch.autograd.grad(b, kg, b.detach())[0], inv(b.detach()))
    a, b = tm.rotary(qg, kg, pos, freq, axes)  # both, but only the key's result is used
    dq, dk = torch.autograd.grad(b.square().sum(), (qg, kg), allow_unused=True)
    assert (dq is None or not dq.any()) and torch.equal(dk, inv(2 * b.detach()))
    shared = _x((2, 1, 5, 32), FP, 25).to(DEV).requires_grad_()  # one head for all
    a, _ = tm.rotary(shared.expand(2, 3, 5, 32), None, pos, freq, axes)
    g = _x((2, 3, 5, 32), FP, 26).to(DEV)
    assert torch.equal(torch.autograd.grad(a, shared, g)[0], inv(g).sum(1, keepdim=True))
    a, _ = tm.rotary(qg, None, pos, freq, axes)
    first, = torch.autograd.grad((a ** 3).sum(), qg, create_graph=True)
    second, = torch.autograd.grad(first.sum(), qg)
    want = inv(6 * a.detach() * tm.rotary(torch.ones_like(q), None, pos, freq, axes)[0])
    assert torch.allclose(second, want, rtol=1e-5, atol=1e-4)


def test_before_attention_in_training():
    """rotary -> F.scaled_dot_product_attention -> backward, against the same in 64 bits on the CPU."""
    B, H, S, D = 1, 4, 70, 64
    freq, axes = tm.rotary_frequencies((8, 12, 12))
    pos = _positions(3, (B, S), 64, 27)
    x = [_x((B, H, S, D), HF, 28 + i) for i in range(4)]
    q, k, v = (t.to(DEV).requires_grad_() for t in x[:3])
    qr, kr = tm.rotary(q, k, pos.to(DEV), freq.to(DEV), axes.to(DEV))
    out = tm.sdpa(qr, kr, v, is_causal=True)
    got = (out,) + torch.autograd.grad(out, (q, k, v), x[3].to(DEV))
    q2, k2, v2 = (t.double().requires_grad_() for t in x[:3])
    s = ref_turn(q2, pos, freq, axes) @ ref_turn(k2, pos, freq, axes).transpose(-1, -2) / 8
    s = s.masked_fill(torch.ones(S, S, dtype=torch.bool).triu(1), float("-inf"))
    o2 = torch.softmax(s, -1) @ v2
    want = (o2,) + torch.autograd.grad(o2, (q2, k2, v2), x[3].double())
    # roundings on the way (turned q and k, probabilities, scores' gradients, outputs), 2^-11 each of values that the largest bounds
    for a, b in zip(got, want):
        assert (a.double().cpu() - b).abs().max() <= 8 * 2.0 ** -11 * max(1.0, float(b.abs().max()))


def ref_turn(x, pos, freq, axes):
    n = len(freq)
    t = torch.stack([pos[int(a)].double() * float(f) for a, f in zip(axes, freq)], -1)[:, None]
    a, b = x[..., :n], x[..., n:]
    return torch.cat([a * t.cos() - b * t.sin(), b * t.cos() + a * t.sin()], -1)


def test_graph():
    freq, axes = (t.to(DEV) for t in tm.rotary_frequencies((8, 24)))
    q = _x((2, 4, 9, 64), BF, 31).to(DEV).requires_grad_()
    k = _x((2, 2, 9, 64), BF, 32).to(DEV).requires_grad_()
    pos, g = _positions(2, (2, 9), 500, 33).to(DEV), _x((2, 4, 9, 64), BF, 34).to(DEV)

    def step():
        a, b = tm.rotary(q, k, pos, freq, axes)
        return (a.detach(), b.detach()) + torch.autograd.grad((a, b), (q, k), (g, g[:, :2]))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(4):
        with torch.no_grad():
            for j, t in enumerate((q, k, g)):
                t.copy_(_x(t.shape, BF, 40 + 3 * i + j))
            pos.copy_(_positions(2, (2, 9), 500, 60 + i))
        want = step()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_nothing_to_turn():
    freq, axes = (t.to(DEV) for t in tm.rotary_frequencies((4,)))
    for shape, p in (((0, 2, 3, 8), (1, 0, 3)), ((2, 2, 0, 8), (1, 0)), ((0, 2, 8), (1, 0))):
        q = torch.zeros(shape, device=DEV, requires_grad=True)
        a, b = tm.rotary(q, q, torch.zeros(p, dtype=torch.int32, device=DEV), freq, axes)
        assert a.shape == b.shape == shape
        assert torch.autograd.grad((a, b), q, (a, b))[0].shape == shape


def test_refusals():
    freq, axes = (t.to(DEV) for t in tm.rotary_frequencies((4,)))
    q = torch.zeros(2, 3, 5, 8, device=DEV)
    pos = torch.zeros(1, 5, dtype=torch.int32, device=DEV)
    ok = dict(query=q, key=q, positions=pos, inv_freq=freq, axes=axes)
    for over, text in ((dict(query=q.double(), key=q.double()), "float32, float16"), (dict(key=q.half()), "same dtype"), (dict(key=q[:, :, :4]), "same tokens"),
                       (dict(query=q[0, 0], key=None), "query must be"), (dict(positions=pos.float()), "int32 or int64"), (dict(positions=pos[:, :4]), "positions must be"),
                       (dict(positions=pos[0]), "positions must be"), (dict(positions=pos.expand(9, 5)), "axes"), (dict(positions=pos[:0]), "axes"),
                       (dict(inv_freq=freq.half()), "float64 or float32"), (dict(axes=axes.long()), "int32"), (dict(axes=axes[:3]), "one entry for each pair"),
                       (dict(inv_freq=freq.repeat(2), axes=axes.repeat(2)), "pairs"), (dict(inv_freq=freq[:0], axes=axes[:0]), "pairs"), (dict(axes=axes.cpu()), "must be on"),
                       (dict(query=q[:, :0], key=None), "no heads")):
        with pytest.raises(RuntimeError, match=text):
            tm.rotary(**{**ok, **over})
