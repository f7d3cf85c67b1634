"""Layer norm kernels (csrc/ln.hip through ops/ln.py) against the formulas in 64
bits.  Tolerances count roundings: U = 2^-24 for each fp32 step -- a sum along a
row is a chain of at most D / 64 + 16 of them --, and half a step of the type
that a result is stored in."""
import copy

import pytest
import torch
import torch.nn.functional as F

from distributed_kfac_pytorch_amd.modules import LayerNorm
from distributed_kfac_pytorch_amd.ops import ln

pytestmark = pytest.mark.gpu

DEV = 'cuda'
U = 2.0 ** -24
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def half(t):
    """(relative, absolute) error of one rounding to type t."""
    return torch.finfo(t).eps / 2, torch.finfo(t).smallest_normal * torch.finfo(t).eps / 2


def make(shape, dtype, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    row = torch.randn(shape[:-1] + (1,), device=DEV, generator=g)
    return (torch.randn(shape, device=DEV, generator=g) * (1 + row.abs()) + row).to(dtype)


def oracle(s, w, b, eps, dy=None, ds=None):
    """Results in 64 bits and the most that each may be off before it is stored."""
    D = s.shape[-1]
    n = D / 64 + 16
    s = s.double().reshape(-1, D)
    w_ = torch.ones(D, dtype=torch.float64, device=s.device) if w is None else w.double()
    b_ = torch.zeros_like(w_) if b is None else b.double()
    d = s - s.mean(1, keepdim=True)
    r = 1 / (d.square().mean(1, keepdim=True) + eps).sqrt()
    h = d * r
    top = s.abs().amax(1, keepdim=True)
    # mean: n roundings of the row's values; variance: n more, and the mean's error squared
    e_mu = n * U * top
    e_r = (n / 2 + 6) * U + (e_mu * r).square()
    e_h = e_mu * r + h.abs() * (e_r + 2 * U)
    out = {'y': (h * w_ + b_, w_.abs() * e_h + 3 * U * ((h * w_).abs() + b_.abs()))}
    if dy is None:
        return out
    dy = dy.double().reshape(-1, D)
    g = dy * w_
    gh = (g * h).mean(1, keepdim=True)
    dx = r * (g - g.mean(1, keepdim=True) - h * gh)
    th = e_h.amax(1, keepdim=True)
    a, ah = g.abs().mean(1, keepdim=True), (g * h).abs().mean(1, keepdim=True)
    e = r * ((n + 8) * U * (g.abs() + a + h.abs() * ah) + e_h * gh.abs() + h.abs() * th * a
             + (g.abs() + a + h.abs() * ah) * e_r)
    if ds is not None:
        dx = dx + ds.double().reshape(-1, D)
        e = e + 2 * U * dx.abs()
    out['dx'] = (dx, e)
    m = min(s.shape[0], 1100) + 16                     # a chain along the rows
    out['dw'] = ((dy * h).sum(0), m * U * (dy * h).abs().sum(0) + (dy.abs() * e_h).sum(0))
    out['db'] = (dy.sum(0), m * U * dy.abs().sum(0))
    return out


def check(name, got, want):
    ref, err = want
    rel, tiny = half(got.dtype)
    off = (got.double().reshape(ref.shape) - ref).abs()
    allow = err + (ref.abs() + err) * rel + tiny
    bad = off > allow
    assert not bad.any() and torch.isfinite(got).all(), \
        (name, int(bad.sum()), float((off / allow).max()))


SHAPES = [(1, 1), (3, 2), (5, 7), (1, 512), (4, 511), (33, 513), (700, 650), (9, 1024),
          (2, 3, 2049), (5, 4097), (3, 8192), (2, 12289), (2, 16384), (2, 16387), (1, 70001),
          (1031, 24), (5000, 40), (2100, 1032), (300, 1), (300, 3), (99, 4), (99, 5), (77, 8), (77, 9)]
TYPES = [(F32, None), (BF16, None), (F16, None), (F32, F32), (BF16, BF16), (F16, F16)]
MIXED = [(F32, BF16), (BF16, F32), (F16, F32), (BF16, F16)]


def run_case(shape, xt, zt, wt='same', bt='same', eps=1e-5, both=True, make_=make):
    x = make_(shape, xt, 1).requires_grad_(True)
    z = None if zt is None else make(shape, zt, 2).requires_grad_(True)
    st = xt if zt is None else torch.promote_types(xt, zt)
    D = shape[-1]
    w = None if wt is None else make((D,), st if wt == 'same' else wt, 3).requires_grad_(True)
    b = None if bt is None else make((D,), st if bt == 'same' else bt, 4).requires_grad_(True)
    assert ln.eligible(x, (D,), w, b, z)
    dy = make(shape, st, 5)
    ds = make(shape, st, 6) if z is not None and both else None
    if z is None:
        y, s = ln.layer_norm(x, D, w, b, eps), x
    else:
        y, s = ln.layer_norm(x, D, w, b, eps, z=z)
        assert s.dtype == st and torch.equal(s, x + z)
    assert y.dtype == st
    torch.autograd.backward([y] if ds is None else [y, s], [dy] if ds is None else [dy, ds])
    o = oracle(s.detach(), w, b, eps, dy, ds)
    check('y', y, o['y'])
    check('dx', x.grad, o['dx'])
    if z is not None:
        # a gradient of the stream's type may be rounded on to z's or x's own
        check('dz', z.grad, o['dx'])
    if w is not None:
        check('dw', w.grad, o['dw'])
    if b is not None:
        check('db', b.grad, o['db'])


@pytest.mark.parametrize('shape', SHAPES)
@pytest.mark.parametrize('xt,zt', TYPES)
def test_forward_and_gradients(shape, xt, zt):
    run_case(shape, xt, zt)


# around the ends of the size classes, more rows than one pass of the workgroups
EDGES = [(2100, 257), (70, 384), (70, 385), (70, 1025), (2100, 1536), (70, 1537), (600, 2500),
         (70, 4096), (1031, 4097), (70, 6144), (70, 6145), (300, 8193), (40, 12288), (530, 12290),
         (9, 16383)]


@pytest.mark.parametrize('shape', EDGES)
@pytest.mark.parametrize('xt,zt', [(F32, F32), (BF16, BF16), (F16, None), (BF16, F32)])
def test_ends_of_the_size_classes(shape, xt, zt):
    run_case(shape, xt, zt)


@pytest.mark.parametrize('shape', [(3, 2), (70, 650), (2, 16387)])
@pytest.mark.parametrize('xt,zt', MIXED)
def test_mixed_streams(shape, xt, zt):
    run_case(shape, xt, zt)


@pytest.mark.parametrize('wt,bt', [(None, None), ('same', None), (None, 'same'), (F32, F32),
                                   (F32, BF16)])
def test_weights_and_types(wt, bt):
    for shape in ((6, 650), (3, 16387)):
        run_case(shape, BF16, BF16, wt, bt)
        run_case(shape, F32, None, wt, bt)


def test_only_the_norm_is_used():
    run_case((40, 96), F32, F32, both=False)


@pytest.mark.parametrize('kind', ['constant', 'offset', 'large', 'tiny'])
@pytest.mark.parametrize('dtype', [F32, BF16])
def test_rows_of_hard_values(kind, dtype):
    def rows(shape, dt, seed):
        if kind == 'constant':
            return torch.full(shape, 3.0, device=DEV, dtype=dt)
        if kind == 'offset':
            return (make(shape, F32, seed) * 0.01 + 1000).to(dt)
        return (make(shape, F32, seed) * (1e15 if kind == 'large' else 1e-10)).to(dt)
    run_case((7, 650), dtype, None, make_=rows)


def test_a_constant_row_is_its_bias():
    """The mean of equal values is that value (sums of up to 2^24 units are exact)."""
    for D in (3, 512, 650, 4097, 20000):
        b = make((D,), F32, 2)
        y = ln.layer_norm(torch.full((4, D), 3.0, device=DEV), D, make((D,), F32, 3), b)
        assert torch.equal(y, b.expand(4, D))


def test_a_bad_row_stays_its_own():
    x = make((6, 130), F32)
    ref = ln.layer_norm(x, 130)
    x[1, 5], x[3, 129], x[4, 0] = float('nan'), float('inf'), float('-inf')
    y = ln.layer_norm(x, 130)
    assert torch.isnan(y[[1, 3, 4]]).all() and torch.equal(y[[0, 2, 5]], ref[[0, 2, 5]])


@pytest.mark.parametrize('dtype', [F32, BF16])
@pytest.mark.parametrize('layout', ['offset', 'sliced', 'every_other', 'transposed', 'expanded',
                                    'one_wide'])
def test_layouts(layout, dtype):
    D = 1 if layout == 'one_wide' else 136
    base = make((12, 300), dtype)
    v = {'offset': lambda: base.flatten()[3:3 + 12 * D].view(12, D),
         'sliced': lambda: base[:, 5:5 + D],
         'every_other': lambda: base[:, ::2][:, :D],
         'transposed': lambda: make((D, 12), dtype).t(),
         'expanded': lambda: base[:1, :D].expand(12, D),
         'one_wide': lambda: base[:, ::7][:, :1]}[layout]()
    x, z = v.detach().requires_grad_(True), v.detach().requires_grad_(True)
    w = make((2 * D,), dtype, 3)[::2].detach().requires_grad_(True)
    dy = v.flip(0) if layout != 'expanded' else make((1, D), dtype, 5).expand(12, D)
    y, s = ln.layer_norm(x, D, w, None, z=z)
    torch.autograd.backward([y, s], [dy, v])
    o = oracle(s.detach(), w, None, 1e-5, dy, v)
    assert torch.equal(s, x + z)
    check('y', y, o['y'])
    for t in (x.grad, z.grad):
        check('dx', t, o['dx'])
    check('dw', w.grad, o['dw'])
    x2 = v.detach().requires_grad_(True)
    ln.layer_norm(x2, D, w).sum().backward()             # a gradient of stride 0
    check('dx', x2.grad, oracle(v, w, None, 1e-5, torch.ones_like(v))['dx'])


def test_broadcast_and_shared_inputs():
    """x used as its own residual, and a broadcast one: autograd sums what each use gives."""
    x = make((4, 6, 64), F32).requires_grad_(True)
    p = make((6, 64), F32, 2).requires_grad_(True)
    y, s = ln.layer_norm(x, 64, z=x)
    dy = make((4, 6, 64), F32, 3)
    y.backward(dy)
    o = oracle((x + x).detach(), None, None, 1e-5, dy)['dx']
    check('dx', x.grad, (2 * o[0], 2 * o[1] + 2 * U * o[0].abs()))
    y, s = ln.layer_norm(x.detach(), 64, z=p.expand(4, 6, 64))
    y.backward(dy)
    o = oracle(s.detach(), None, None, 1e-5, dy)['dx']
    per = [t.reshape(4, 6, 64).sum(0) for t in o]
    check('dp', p.grad, (per[0], per[1] + 8 * U * o[0].abs().reshape(4, 6, 64).sum(0)))


def test_frozen_parts():
    """Gradients that nobody asks for are not computed, the others stay the same."""
    x, dy = make((50, 72), F32), make((50, 72), F32, 2)
    w, b = make((72,), F32, 3), make((72,), F32, 4)

    def grads(mask):
        t = [v.clone().requires_grad_(m) for v, m in zip((x, w, b, x), mask)]
        y, s = ln.layer_norm(t[0], 72, t[1], t[2], z=t[3])
        y.backward(dy)
        return [v.grad for v in t]
    full = grads((True, True, True, True))
    for mask in ((True, False, False, False), (False, True, False, False),
                 (False, False, True, False), (False, False, False, True)):
        for g, f, m in zip(grads(mask), full, mask):
            assert (g is None) == (not m) and (g is None or torch.equal(g, f))
    t = x.clone().requires_grad_(True)
    y, s = ln.layer_norm(t, 72, z=x)
    assert torch.equal(torch.autograd.grad(s, t, dy)[0], dy)      # the sum alone is used


def test_no_rows():
    x = torch.empty(0, 8, device=DEV, requires_grad=True)
    w = torch.ones(8, device=DEV, requires_grad=True)
    y, s = ln.layer_norm(x, 8, w, z=x)
    y.sum().backward()
    assert y.shape == (0, 8) and torch.equal(w.grad, torch.zeros_like(w))


@pytest.mark.parametrize('dtype', [F32, BF16])
def test_difference_quotient(dtype):
    """The gradient along a direction against the function's own values.  fp32
    results of 800 rows differ from the real function by about U a value, over a
    step of 2^-5: 1e-3 of the slope is far above both that and the third
    derivative's h^2."""
    x, v, c = (make((80, 96), dtype, k).float() for k in (1, 2, 3))
    v, c = v / v.std(), c / c.std()
    w = make((96,), F32, 4)
    h = 2.0 ** -5

    def f(t):
        return (ln.layer_norm(t, 96, w).double() * c.double()).sum()
    xg = x.clone().requires_grad_(True)
    ln.layer_norm(xg, 96, w).backward(c)
    slope = (xg.grad.double() * v.double()).sum()
    scale = xg.grad.double().norm() * v.double().norm()
    diff = (f(x + h * v) - f(x - h * v)) / (2 * h)
    assert abs(float(diff - slope)) < 2e-3 * float(scale)


def test_second_derivative_is_torchs():
    x, w, b = make((9, 40), F32).requires_grad_(True), make((40,), F32, 2).requires_grad_(True), \
        make((40,), F32, 3).requires_grad_(True)

    def gg(f, *xs):
        xs = [t.detach().double().requires_grad_(True) if f is None else
              t.detach().requires_grad_(True) for t in xs]
        if f is None:
            s = xs[0] + xs[0].cos()
            y = F.layer_norm(s, (40,), xs[1], xs[2])
        else:
            y, s = f(xs[0], xs[1], xs[2])
        g = torch.autograd.grad((y.sin() + s.square()).sum(), xs, create_graph=True)
        return torch.autograd.grad(sum(t.square().sum() for t in g), xs)
    ours = gg(lambda x, w, b: ln.layer_norm(x, 40, w, b, z=x.cos()), x, w, b)
    ref = gg(None, x, w, b)
    for a, r in zip(ours, ref):
        assert float((a.double() - r).norm() / r.norm()) < 1e-4      # ~1e3 fp32 steps deep


def test_autocast_keeps_fp32():
    x, w = make((10, 64), BF16).requires_grad_(True), make((64,), F32, 2).requires_grad_(True)
    with torch.autocast('cuda', dtype=BF16):
        y = ln.layer_norm(x, 64, w)
        r = F.layer_norm(x.detach(), (64,), w.detach())
    assert y.dtype == r.dtype == F32
    dy = make((10, 64), F32, 3)
    y.backward(dy)
    o = oracle(x.detach(), w, None, 1e-5, dy)
    check('y', y, o['y'])
    check('dx', x.grad, o['dx'])
    check('dw', w.grad, o['dw'])


@pytest.mark.parametrize('rows,D,dtype', [(700, 650, F32), (300, 2048, BF16), (3, 16387, F32)])
def test_bitwise_repeatable_and_captured(rows, D, dtype):
    """Twice the same bits, on another stream too; a captured step replays them
    for new inputs, with eager work between the replays."""
    mod = LayerNorm(D, device=DEV, dtype=dtype)
    x, z, dy, ds = (make((rows, D), dtype, k) for k in range(4))

    def step(x, z, m):
        x, z = x.detach().requires_grad_(True), z.detach().requires_grad_(True)
        y, s = m(x, z)
        return (y.detach(), s.detach()) + torch.autograd.grad(
            [y, s], [x, z, m.weight, m.bias], [dy, ds])
    first = step(x, z, mod)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = step(x, z, mod)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(first, again))
    m2 = copy.deepcopy(mod)
    xs, zs = x.clone(), z.clone()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step(xs, zs, m2)
    for k in range(3):
        xs.copy_(make((rows, D), dtype, 10 + k))
        ref = step(xs, zs, mod)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, ref)), k


@pytest.mark.parametrize('D', [64, 20000])
def test_offsets_past_32_bits(D):
    """The last rows of more than 2^31 elements, 2^32 bytes."""
    rows = 2 ** 31 // D + 5
    x = torch.zeros(rows, D, dtype=BF16, device=DEV)
    x[-3:] = make((3, D), BF16)
    x.requires_grad_(True)
    w = make((D,), BF16, 2).requires_grad_(True)
    y = ln.layer_norm(x, D, w)
    dy = torch.zeros_like(y)
    dy[-3:] = make((3, D), BF16, 3)
    dx, dw = torch.autograd.grad(y, [x, w], dy)
    o = oracle(x.detach()[-3:], w, None, 1e-5, dy[-3:])
    check('y', y[-3:], o['y'])
    check('dx', dx[-3:], o['dx'])
    check('dw', dw, o['dw'])
    assert not y[:-3].any() and not dx[:-3].any()


def test_traces_and_modes_see_torch():
    """A trace of the module and a dispatch mode around it hold torch's own norm."""
    from torch.utils._python_dispatch import TorchDispatchMode
    m = LayerNorm(32, device=DEV)
    x, x2 = make((4, 32), F32), make((4, 32), F32, 2)
    t = torch.jit.trace(m, (x,))
    check('trace', t(x2), oracle(x2, None, None, 1e-5)['y'])
    seen = []

    class Mode(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            seen.append(str(func))
            return func(*args, **(kwargs or {}))
    with Mode():
        m(x)
    assert any('layer_norm' in s for s in seen)


def test_module_switch(monkeypatch):
    x = make((4, 32), F32)
    m = LayerNorm(32, device=DEV)
    y = m(x)
    monkeypatch.setattr(ln, 'ENABLED', False)
    assert not ln.eligible(x, (32,))
    check('y', m(x), oracle(x, None, None, 1e-5)['y'])
    check('y', y, oracle(x, None, None, 1e-5)['y'])


@pytest.mark.parametrize('transform', ['grad', 'vmap', 'jvp'])
def test_transforms_reach_torch(transform):
    x, w = make((3, 8), F32), make((8,), F32, 2)

    def f(t):
        return ln.layer_norm(t, 8, w).square().sum()

    def ref(t):
        return F.layer_norm(t, (8,), w).square().sum()
    if transform == 'grad':
        a, b = torch.func.grad(f)(x), torch.func.grad(ref)(x)
    elif transform == 'vmap':
        a, b = torch.func.vmap(f)(x), torch.func.vmap(ref)(x)
    else:
        a, b = torch.func.jvp(f, (x,), (x,))[1], torch.func.jvp(ref, (x,), (x,))[1]
    assert torch.equal(a, b)
