"""GPU: the learned-appearance operators (tidegs_b200.appearance) against
their 64-bit oracle (oracle/appearance.py).

Tolerances are worst-case rounding bounds, carried through the formulas next
to the values (class V): every product of K terms may be off by (K + 2) u
times the product of the magnitudes, with u = 2^-23 (twice a 32-bit rounding,
so that a sum which truncates is covered), every stored value by half a step
of its type (bf16 2^-8, fp16 2^-11, fp32 2^-24, relative). Dropout is exact:
one 32-bit product, one rounding."""
import math

import numpy as np
import pytest
import torch

from oracle import appearance as orc

pytestmark = pytest.mark.gpu

U = 2.0 ** -23
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
# smallest magnitude that keeps the relative step (below it, steps are absolute)
TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -25}
TYPES = [torch.float32, torch.bfloat16, torch.float16]


class V:
    """A 64-bit value and a bound on how far the kernel's may be from it."""

    def __init__(self, val, err=None):
        self.val = val.double()
        self.err = torch.zeros_like(self.val) if err is None else err

    @property
    def most(self):
        return self.val.abs() + self.err

    def __matmul__(self, o):
        k = self.val.shape[-1]
        err = self.err @ o.val.abs() + self.val.abs() @ o.err + self.err @ o.err
        return V(self.val @ o.val, err + (k + 2) * U * (self.most @ o.most))

    def __mul__(self, o):
        err = self.err * o.val.abs() + self.val.abs() * o.err + self.err * o.err
        return V(self.val * o.val, err + U * self.most * o.most)

    def __add__(self, o):
        return V(self.val + o.val, self.err + o.err + U * (self.most + o.most))

    @property
    def T(self):
        return V(self.val.T, self.err.T)

    def stored(self, dtype):
        return V(self.val, self.err + HALF[dtype] * self.most + TINY[dtype])


def _far(got, want: V, what):
    got = got.detach().double()
    assert got.shape == want.val.shape, what
    bad = (got - want.val).abs() > want.err
    if bool(bad.any()) or not bool(torch.isfinite(got).all()):
        i = int(((got - want.val).abs() / want.err.clamp_min(1e-300)).flatten().argmax())
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} values are off; worst at {i}: "
                             f"{got.flatten()[i]:.9g} for {want.val.flatten()[i]:.9g}, bound "
                             f"{want.err.flatten()[i]:.3g}")


def _rand(g, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


# --- layer norm --------------------------------------------------------------

def _norm_inputs(n, c, dtype, ptype, seed=0):
    g = _gen(seed)
    x = torch.randn(n, c, generator=g, device="cuda") * (0.5 + torch.rand(n, 1, generator=g, device="cuda"))
    x = (x + torch.randn(n, 1, generator=g, device="cuda")).to(dtype)
    return (x, (1 + 0.2 * torch.randn(c, generator=g, device="cuda")).to(ptype),
            _rand(g, c, dtype=ptype, scale=0.3), _rand(g, n, c, dtype=dtype, scale=0.1))


def _norm_expect(x, w, b, eps, v, dtype, ptype):
    """(y, v_x, v_w, v_b) with bounds. A row's sums have c terms of up to
    amax; z inherits (amax / std) times the unit from the mean's subtraction,
    and the spread's relative error is of the same size."""
    x, v = x.double(), v.double()
    w64 = torch.ones_like(x[0]) if w is None else w.double()
    b64 = torch.zeros_like(x[0]) if b is None else b.double()
    n, c = x.shape
    d = x - x.mean(1, keepdim=True)
    std = torch.sqrt((d * d).mean(1, keepdim=True) + eps)
    unit = (c + 16) * U * (1 + x.abs().amax(1, keepdim=True) / std)
    z = V(d / std, unit * (1 + (d / std).abs()))
    y = (z * V(w64) + V(b64.expand(n, c))).stored(dtype)
    want = [y]
    g = V(v) * V(w64)
    m1 = V(g.val.mean(1, keepdim=True), g.err.mean(1, keepdim=True)
           + (c + 2) * U * g.most.mean(1, keepdim=True))
    gz = g * z
    m2 = V(gz.val.mean(1, keepdim=True), gz.err.mean(1, keepdim=True)
           + (c + 2) * U * gz.most.mean(1, keepdim=True))
    inner = g + V(-m1.val, m1.err) + V(-z.val, z.err) * m2
    rstd = V(1 / std, unit / std)
    want.append((rstd * inner).stored(dtype))
    vz = V(v) * z
    want.append(V(vz.val.sum(0), vz.err.sum(0) + (n + 2) * U * vz.most.sum(0)).stored(ptype))
    want.append(V(v.sum(0), (n + 2) * U * v.abs().sum(0)).stored(ptype))
    return want


def _norm_check(x, w, b, v, eps=1e-5):
    from tidegs_b200 import appearance as ap

    dtype = x.dtype
    ptype = w.dtype if w is not None else b.dtype if b is not None else dtype
    leaves = [t.detach().requires_grad_(True) if t is not None else None for t in (x, w, b)]
    y = ap.layer_norm(*leaves, eps)
    assert y.dtype == dtype
    grads = torch.autograd.grad(y, [t for t in leaves if t is not None], v)
    want = _norm_expect(x, w, b, eps, v, dtype, ptype)
    _far(y, want[0], "y")
    with torch.no_grad():
        assert torch.equal(ap.layer_norm(x, w, b, eps), y)
    names = [k for k, t in zip(("v_x", "v_w", "v_b"), leaves) if t is not None]
    expect = [e for e, t in zip(want[1:], leaves) if t is not None]
    for name, got, e in zip(names, grads, expect):
        _far(got, e, name)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,c", [(1, 1), (1, 64), (3, 2), (257, 3), (130, 7), (64, 8), (1000, 16),
                                 (777, 31), (500, 32), (333, 48), (2049, 59), (1500, 64), (129, 100),
                                 (70, 127), (65, 128), (40, 129), (33, 255), (50, 256), (21, 500),
                                 (19, 512), (18, 516), (9, 768), (7, 1000), (5, 1024), (4, 1025),
                                 (3, 2048), (2, 2056), (3, 5000), (2, 8191), (2, 8192)])
def test_layer_norm(dtype, n, c):
    _norm_check(*_norm_inputs(n, c, dtype, dtype))


@pytest.mark.parametrize("dtype", TYPES)
def test_layer_norm_many_rows(dtype):
    # more rows than one sweep of the grid takes, and a ragged last tile
    _norm_check(*_norm_inputs(50001, 24, dtype, dtype))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_layer_norm_parameters_in_32_bits(dtype):
    x, w, b, v = _norm_inputs(300, 40, dtype, torch.float32)
    _norm_check(x, w, b, v)
    _norm_check(x, None, b, v)
    _norm_check(x, w, None, v)
    _norm_check(x, None, None, v)


@pytest.mark.parametrize("dtype", TYPES)
def test_layer_norm_strides_and_alignment(dtype):
    g = _gen(5)
    wide = _rand(g, 64, 100, dtype=dtype)
    vwide = _rand(g, 64, 100, dtype=dtype, scale=0.1)
    w, b = _rand(g, 32, dtype=dtype), _rand(g, 32, dtype=dtype)
    for cols in (slice(0, 32), slice(1, 33), slice(8, 40), slice(0, 64, 2)):
        _norm_check(wide[:, cols], w, b, vwide[:, cols])
    _norm_check(wide[::2, 4:36], w[:], b, vwide[1::2, :32])
    _norm_check(wide[:32].T[:32, :].T, w, b, vwide[:32, :32])  # columns of another stride
    from tidegs_b200 import appearance as ap

    x3 = _rand(g, 3, 5, 32, dtype=dtype)
    assert torch.equal(ap.layer_norm(x3, w, b), ap.layer_norm(x3.reshape(15, 32), w, b).reshape(3, 5, 32))
    one = _rand(g, 32, dtype=dtype)
    assert torch.equal(ap.layer_norm(one, w, b), ap.layer_norm(one[None], w, b)[0])


def test_layer_norm_edges():
    from tidegs_b200 import appearance as ap

    x = torch.empty(0, 16, device="cuda", requires_grad=True)
    w = torch.ones(16, device="cuda", requires_grad=True)
    b = torch.zeros(16, device="cuda", requires_grad=True)
    y = ap.layer_norm(x, w, b)
    assert y.shape == (0, 16)
    for t in torch.autograd.grad(y.sum(), (x, w, b)):
        assert not t.any()
    # a constant row: z = 0; a row with NaN or infinity poisons itself alone
    x = torch.full((4, 16), 3.0, device="cuda")
    x[1, 2], x[2, 3] = float("nan"), float("inf")
    y = ap.layer_norm(x, None, b.detach() + 2)
    assert torch.all(y[0] == 2) and torch.all(y[3] == 2) and torch.isnan(y[1]).all() and torch.isnan(y[2]).all()
    # a gradient of stride zero (the sum's)
    x = _rand(_gen(1), 6, 16).requires_grad_(True)
    _far(torch.autograd.grad(ap.layer_norm(x, w, b).sum(), x)[0],
         _norm_expect(x.detach(), w.detach(), b.detach(), 1e-5, torch.ones(6, 16, device="cuda"),
                      torch.float32, torch.float32)[1], "v_x")


def test_layer_norm_partial_gradients_agree():
    from tidegs_b200 import appearance as ap

    x, w, b, v = _norm_inputs(700, 59, torch.float32, torch.float32)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    full = torch.autograd.grad(ap.layer_norm(*leaves), leaves, v)
    for k in range(3):
        part = [t.detach().requires_grad_(i == k) for i, t in enumerate(leaves)]
        assert torch.equal(torch.autograd.grad(ap.layer_norm(*part), part[k], v)[0], full[k])


# --- gated feed-forward block --------------------------------------------------

def _ffn_inputs(n, d, h, o, dtype, seed=0):
    g = _gen(seed)
    return (_rand(g, n, d, dtype=dtype), _rand(g, h, d, dtype=dtype, scale=d ** -0.5),
            _rand(g, h, d, dtype=dtype, scale=d ** -0.5), _rand(g, o, h, dtype=dtype, scale=h ** -0.5),
            _rand(g, n, o, dtype=dtype, scale=0.1))


def _ffn_expect(x, wg, wu, wd, v, dtype, parts=1):
    """`parts`: bf16 parts of a hidden value; the last leaves half its step, 2^-8
    of what the others left."""
    x, wg, wu, wd, v = (V(t) for t in (x, wg, wu, wd, v))
    hid = (lambda t: V(t.val, t.err + HALF[dtype] ** parts * t.most + TINY[dtype])) \
        if dtype == torch.bfloat16 else (lambda t: t)
    g, u = x @ wg.T, x @ wu.T
    # exp and the quotient: a few steps, and one per unit of the exponent
    wave = (16 + 2 * g.most) * U
    act = V(orc.silu(g.val), 1.1 * g.err + wave * orc.silu(g.val).abs())
    slope = V(orc.silu_slope(g.val), 0.5 * g.err + wave * (1 + g.most))
    hh = act * u
    y = (hid(hh) @ wd.T).stored(dtype)
    vh = v @ wd
    vu, vg = hid(vh * act), hid(vh * u * slope)
    return dict(y=y, v_x=(vg @ wg + vu @ wu).stored(dtype), v_w_gate=(vg.T @ x).stored(dtype),
                v_w_up=(vu.T @ x).stored(dtype), v_w_down=(v.T @ hid(hh)).stored(dtype))


def _ffn_check(x, wg, wu, wd, v):
    from tidegs_b200 import appearance as ap

    leaves = [t.detach().requires_grad_(True) for t in (x, wg, wu, wd)]
    y = ap.gated_feed_forward(*leaves)
    grads = torch.autograd.grad(y, leaves, v)
    want = _ffn_expect(x, wg, wu, wd, v, x.dtype)
    for (name, e), got in zip(want.items(), (y, *grads)):
        assert got.dtype == x.dtype
        _far(got, e, name)
    with torch.no_grad():
        assert torch.equal(ap.gated_feed_forward(x, wg, wu, wd), y)
    again = torch.autograd.grad(ap.gated_feed_forward(*leaves), leaves, v)
    for a, e in zip(again, grads):
        assert torch.equal(a, e)


FFN_SIZES = [(1, 1, 1, 1), (1, 32, 64, 3), (2, 3, 5, 2), (31, 8, 16, 3), (32, 16, 16, 16),
             (33, 17, 33, 19), (127, 32, 64, 3), (128, 64, 128, 48), (129, 64, 128, 48),
             (255, 59, 100, 59), (500, 35, 96, 3), (300, 128, 256, 128), (200, 200, 40, 30),
             (200, 24, 40, 200), (130, 256, 512, 256), (140, 255, 130, 255), (64, 64, 1000, 64),
             (1000, 8, 48, 3), (40, 16, 4096, 8), (257, 96, 192, 65), (257, 65, 65, 129),
             (2000, 48, 80, 48), (384, 128, 384, 128), (150, 144, 320, 160)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,d,h,o", FFN_SIZES)
def test_gated_feed_forward(dtype, n, d, h, o):
    _ffn_check(*_ffn_inputs(n, d, h, o, dtype))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,d,h,o", [(40003, 32, 64, 3), (30011, 64, 128, 48), (20000, 128, 160, 96),
                                     (60000, 256, 192, 256), (50000, 130, 129, 200), (60000, 200, 100, 16),
                                     (60000, 16, 60, 256), (60000, 33, 64, 35)])
def test_gated_feed_forward_many_rows(dtype, n, d, h, o):
    _ffn_check(*_ffn_inputs(n, d, h, o, dtype))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_gated_feed_forward_strides_and_alignment(dtype):
    x, wg, wu, wd, v = _ffn_inputs(150, 96, 64, 96, dtype)
    for cols in (slice(0, 32), slice(1, 33), slice(8, 40), slice(5, 64), slice(0, 64, 2)):
        _ffn_check(x[:, cols], wg[:, cols], wu[:, cols], wd[cols], v[:, cols])
    _ffn_check(x[::3], wg, wu, wd, v[::3])
    _ffn_check(x[:96].T.contiguous().T, wg, wu, wd, v[:96])
    _ffn_check(x, wg, wu, wd.T.contiguous().T, v)
    from tidegs_b200 import appearance as ap

    y = ap.gated_feed_forward(x.reshape(5, 30, 96), wg, wu, wd)
    assert torch.equal(y.reshape(150, 96), ap.gated_feed_forward(x, wg, wu, wd))
    assert torch.equal(ap.gated_feed_forward(x[7], wg, wu, wd), y.reshape(150, 96)[7])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_gated_feed_forward_edges(dtype):
    from tidegs_b200 import appearance as ap

    x, wg, wu, wd, v = (t.requires_grad_(True) for t in _ffn_inputs(200, 40, 72, 24, dtype))
    none = x[:0]
    y = ap.gated_feed_forward(none, wg, wu, wd)
    assert y.shape == (0, 24)
    for t in torch.autograd.grad(y.sum(), (wg, wu, wd)):
        assert not t.any()
    # rows that hold NaN or infinity stay alone
    clean = ap.gated_feed_forward(x, wg, wu, wd).detach()
    bad = x.detach().clone()
    bad[3, 5], bad[150, 0] = float("nan"), float("inf")
    y = ap.gated_feed_forward(bad, wg, wu, wd)
    keep = [i for i in range(200) if i not in (3, 150)]
    assert torch.equal(y[keep], clean[keep]) and torch.isnan(y[3]).all()
    # gates far from zero: silu is 0 on the left, the identity on the right
    big = torch.zeros(2, 40, device="cuda", dtype=dtype)
    big[0, 0], big[1, 0] = 1000.0, -1000.0
    one = torch.zeros(72, 40, device="cuda", dtype=dtype)
    one[0, 0] = 1.0
    down = torch.ones(24, 72, device="cuda", dtype=dtype)
    want = torch.tensor([[1e6], [0.0]], device="cuda", dtype=dtype).expand(2, 24)
    leaves = [t.requires_grad_(True) for t in (big, one, one.clone(), down)]
    y = ap.gated_feed_forward(*leaves)
    assert torch.equal(y, want)
    grads = torch.autograd.grad(y, leaves, torch.ones_like(y))
    assert all(bool(torch.isfinite(t).all()) for t in grads)
    # d(g^2)/dx at g = x = 1000, summed over 24 outputs; zero on the left
    exact = torch.tensor([24 * 2000.0, 0.0], dtype=torch.float64, device="cuda")
    assert bool(((grads[0][:, 0].double() - exact).abs() <= 4 * HALF[dtype] * exact).all())


def test_gated_feed_forward_partial_gradients_agree():
    from tidegs_b200 import appearance as ap

    for dtype in (torch.float32, torch.bfloat16):
        *ins, v = _ffn_inputs(600, 64, 128, 48, dtype)
        leaves = [t.requires_grad_(True) for t in ins]
        full = torch.autograd.grad(ap.gated_feed_forward(*leaves), leaves, v)
        for k in range(4):
            part = [t.detach().requires_grad_(i == k) for i, t in enumerate(leaves)]
            assert torch.equal(torch.autograd.grad(ap.gated_feed_forward(*part), part[k], v)[0], full[k])


@pytest.mark.parametrize("n,d,h,o", [(1, 35, 96, 3), (40, 10, 24, 88), (500, 145, 72, 9),
                                     (1500, 32, 64, 3), (700, 192, 300, 128), (300, 256, 500, 256)])
def test_small_bfloat16_calls_round_once(n, d, h, o):
    """A call of one tile per SM keeps hidden values in two bf16 parts."""
    from tidegs_b200 import appearance as ap

    *ins, v = _ffn_inputs(n, d, h, o, torch.bfloat16, 3)
    leaves = [t.requires_grad_(True) for t in ins]
    y = ap.gated_feed_forward(*leaves)
    grads = torch.autograd.grad(y, leaves, v)
    want = _ffn_expect(*(t.detach() for t in ins), v, torch.bfloat16, parts=2)
    for (name, e), got in zip(want.items(), (y, *grads)):
        _far(got, e, name)


def test_gated_feed_forward_gradient_matches_differences():
    """Directional derivatives of the 32-bit kernel against central
    differences of its own forward: step e leaves e^2 / 6 times the third
    derivative, and each loss its forward's rounding over e."""
    from tidegs_b200 import appearance as ap

    *ins, v = _ffn_inputs(64, 24, 48, 8, torch.float32)
    leaves = [t.requires_grad_(True) for t in ins]
    y = ap.gated_feed_forward(*leaves)
    grads = torch.autograd.grad(y, leaves, v)
    e = 2.0 ** -6
    for k, t in enumerate(ins):
        step = _rand(_gen(k + 9), *t.shape)
        step = step / step.norm() * math.sqrt(t.shape[0])

        def loss(s, exact):
            moved = [p.detach() + s * step if i == k else p.detach() for i, p in enumerate(ins)]
            f = orc.gated_feed_forward if exact else ap.gated_feed_forward
            moved = [m.double() for m in moved] if exact else moved
            return (f(*moved).double() * v.double()).sum()

        want = float((grads[k].double() * step.double()).sum())
        got = float((loss(e, False) - loss(-e, False)) / (2 * e))
        # the truncation term, from the oracle at two steps (Richardson)
        d1 = float((loss(e, True) - loss(-e, True)) / (2 * e))
        d2 = float((loss(e / 2, True) - loss(-e / 2, True)) / e)
        rounding = float(_ffn_expect(*[p.detach() for p in ins], v, torch.float32)["y"].err.mul(
            v.double().abs()).sum()) / e
        assert abs(got - want) <= 2 * abs(d1 - d2) * 4 / 3 + 2 * rounding


# --- dropout -------------------------------------------------------------------

def _drop_expect(x, p, keep):
    scale = np.float32(1.0 / (1.0 - p)) if p < 1 else np.float32(0)
    y = x.float() * torch.tensor(scale, device=x.device)
    return torch.where(keep, y, torch.zeros((), device=x.device)).to(x.dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,c", [(1, 1), (5, 1), (4097, 1), (100, 2), (1000, 3), (77, 4), (501, 5),
                                 (300, 8), (129, 27), (2000, 48), (4001, 64), (33, 100), (40, 257),
                                 (3, 4096), (2, 65535), (2, 65536)])
@pytest.mark.parametrize("per_row", [False, True])
def test_dropout_is_exact(dtype, n, c, per_row):
    from tidegs_b200 import appearance as ap

    g = _gen(n + c)
    x = _rand(g, n, c, dtype=dtype).requires_grad_(True)
    v = _rand(g, n, c, dtype=dtype, scale=0.1)
    ids = torch.randint(-2 ** 40, 2 ** 40, (n,), generator=g, device="cuda")
    for p, seed, offset, who in ((0.3, 2 ** 63 + 17, 9, None), (0.75, 5, 2 ** 32 - 1, ids)):
        y = ap.dropout(x, p, seed, offset=offset, ids=who, per_row=per_row)
        keep = torch.from_numpy(orc.dropout_keep(n, c, p, seed, offset,
                                                 None if who is None else who.cpu().numpy(),
                                                 per_row)).cuda()
        assert torch.equal(y, _drop_expect(x.detach(), p, keep))
        assert torch.equal(torch.autograd.grad(y, x, v)[0], _drop_expect(v, p, keep))


def test_dropout_ends_and_masked_values():
    from tidegs_b200 import appearance as ap

    x = _rand(_gen(0), 300, 12)
    assert torch.equal(ap.dropout(x, 0.0, 3), x)
    assert not ap.dropout(x, 1.0, 3).any()
    keep = torch.from_numpy(orc.dropout_keep(300, 12, 0.5, 3)).cuda()
    bad = torch.where(keep, x, torch.full_like(x, float("nan")))
    assert torch.equal(ap.dropout(bad, 0.5, 3), _drop_expect(x, 0.5, keep))
    bad = torch.where(keep, x, torch.full_like(x, float("inf")))
    assert torch.equal(ap.dropout(bad, 0.5, 3), _drop_expect(x, 0.5, keep))
    assert ap.dropout(x[:0], 0.5, 3).shape == (0, 12)
    # the share that is kept: 6 standard deviations of a fair coin
    big = ap.dropout(torch.ones(1 << 20, device="cuda"), 0.5, 77)
    assert abs(int((big > 0).sum()) - (1 << 19)) < 6 * 512


@pytest.mark.parametrize("dtype", TYPES)
def test_dropout_strides_shapes_and_ids(dtype):
    from tidegs_b200 import appearance as ap

    wide = _rand(_gen(2), 90, 64, dtype=dtype)
    for x in (wide[:, 8:40], wide[:, 1:33], wide[::2, :32], wide[:, ::2], wide.T, wide[:1].expand(90, 64)):
        assert torch.equal(ap.dropout(x, 0.4, 8, offset=2), ap.dropout(x.contiguous(), 0.4, 8, offset=2))
    x3 = wide.reshape(90, 16, 4)
    assert torch.equal(ap.dropout(x3, 0.4, 8).reshape(90, 64), ap.dropout(wide, 0.4, 8))
    x1 = wide[:, 3]
    assert torch.equal(ap.dropout(x1, 0.4, 8), ap.dropout(x1.reshape(90, 1), 0.4, 8)[:, 0])
    # a Gaussian keeps its draw wherever its row is, also twice in one call
    ids = torch.arange(90, device="cuda") * 3 + 2 ** 33
    pick = torch.tensor([5, 5, 80, 0, 5], device="cuda")
    full = ap.dropout(wide, 0.4, 8, ids=ids)
    assert torch.equal(ap.dropout(wide[pick], 0.4, 8, ids=ids[pick]), full[pick])
    assert torch.equal(ap.dropout(wide[::3], 0.4, 8, ids=ids[::3]), full[::3])


def test_dropout_offset_on_the_device():
    from tidegs_b200 import appearance as ap

    x = _rand(_gen(4), 500, 20).requires_grad_(True)
    step = torch.tensor([6], device="cuda")
    y = ap.dropout(x, 0.5, 1, offset=step)
    assert torch.equal(y, ap.dropout(x, 0.5, 1, offset=6))
    step += 1  # between a call and its backward: refused
    with pytest.raises(RuntimeError, match="inplace"):
        torch.autograd.grad(y, x, torch.ones_like(y))


# --- streams, graphs, together ---------------------------------------------------

def test_operators_follow_the_current_stream():
    from tidegs_b200 import appearance as ap

    *ins, v = _ffn_inputs(4000, 64, 128, 48, torch.bfloat16)
    want = ap.dropout(ap.gated_feed_forward(ap.layer_norm(ins[0]), *ins[1:]), 0.2, 4)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        torch.cuda._sleep(2_000_000)
        x = torch.zeros_like(ins[0])
        x.copy_(ins[0])
        got = ap.dropout(ap.gated_feed_forward(ap.layer_norm(x), *ins[1:]), 0.2, 4)
    side.synchronize()
    assert torch.equal(got, want)


def test_operators_capture_and_replay():
    """A training step captured once and replayed on new inputs and steps."""
    from tidegs_b200 import appearance as ap

    *ins, v = _ffn_inputs(3000, 32, 64, 16, torch.bfloat16)
    x, wg, wu, wd = (t.requires_grad_(True) for t in ins)
    nw = torch.ones(32, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    step = torch.zeros(1, dtype=torch.int64, device="cuda")

    def train():
        y = ap.dropout(ap.gated_feed_forward(ap.layer_norm(x, nw), wg, wu, wd), 0.3, 21, offset=step)
        return (y.detach(), *torch.autograd.grad(y, (x, nw, wg, wu, wd), v))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        train()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = train()
    for k in range(3):
        with torch.no_grad():
            x.copy_(_rand(_gen(100 + k), 3000, 32, dtype=torch.bfloat16))
        step.fill_(k)
        graph.replay()
        for a, e in zip(held, train()):
            assert torch.equal(a, e)


def test_two_streams_at_once():
    """Two training steps enqueued on two streams share nothing."""
    from tidegs_b200 import appearance as ap

    def job(seed):
        *ins, v = _ffn_inputs(20000, 64, 128, 48, torch.bfloat16, seed)
        return [t.requires_grad_(True) for t in ins], v

    def train(leaves, v):
        y = ap.gated_feed_forward(ap.layer_norm(leaves[0]), *leaves[1:])
        return torch.autograd.grad(y, leaves, v)

    jobs = [job(1), job(2)]
    want = [train(*j) for j in jobs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(5):
        for k in (0, 1):
            with torch.cuda.stream(streams[k]):
                got[k].append(train(*jobs[k]))
    torch.cuda.synchronize()
    for k in (0, 1):
        for g in got[k]:
            for a, e in zip(g, want[k]):
                assert torch.equal(a, e)


@pytest.mark.parametrize("dtype,n,d,h,o", [(torch.float32, 9000, 128, 192, 64),
                                           (torch.float32, 9000, 24, 48, 16),
                                           (torch.bfloat16, 9000, 35, 100, 3),
                                           (torch.bfloat16, 9000, 160, 320, 192)])
def test_gated_feed_forward_captured_and_on_two_streams(dtype, n, d, h, o):
    """Each of the block's kernels: a training step enqueued on two streams at
    once, and one captured and replayed on other inputs."""
    from tidegs_b200 import appearance as ap

    def job(seed):
        *ins, v = _ffn_inputs(n, d, h, o, dtype, seed)
        return [t.requires_grad_(True) for t in ins], v

    def train(leaves, v):
        y = ap.gated_feed_forward(*leaves)
        return (y.detach(), *torch.autograd.grad(y, leaves, v))

    jobs = [job(1), job(2)]
    want = [train(*j) for j in jobs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(3):
        for k in (0, 1):
            with torch.cuda.stream(streams[k]):
                got[k].append(train(*jobs[k]))
    torch.cuda.synchronize()
    for k in (0, 1):
        for g in got[k]:
            for a, e in zip(g, want[k]):
                assert torch.equal(a, e)
    leaves, v = jobs[0]
    del got
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = train(leaves, v)
    with torch.no_grad():
        for t, other in zip(leaves, jobs[1][0]):
            t.copy_(other)
        v.copy_(jobs[1][1])
    graph.replay()
    for a, e in zip(held, want[1]):
        assert torch.equal(a, e)
    ap.check()


@pytest.mark.parametrize("n,c", [(1, 1), (3, 7), (1000, 3), (129, 35), (70, 64), (33, 255)])
def test_align_rows(n, c):
    from tidegs_b200 import _lib

    wide = _rand(_gen(3), n, c + 5, dtype=torch.bfloat16)
    for src in (wide[:, :c].contiguous(), wide[:, 1:c + 1]):
        units = -(-c // 8) * 8
        out = torch.full((n, units), 7.0, dtype=torch.bfloat16, device="cuda")
        _lib.call("tgs_align_rows", src.data_ptr(), src.stride(0) if n > 1 else c, n, c, out.data_ptr(),
                  torch.cuda.current_stream().cuda_stream)
        assert torch.equal(out[:, :c], src) and not out[:, c:].any()


def test_check_reads_the_error_word():
    """A wait that ran out is told by check() (the word is set by hand)."""
    from tidegs_b200 import appearance as ap

    *ins, _ = _ffn_inputs(10, 16, 16, 16, torch.bfloat16)
    ap.gated_feed_forward(*ins)
    ap.check()
    ap.check("cuda")
    word = ap._err_words[ins[0].device]
    word[0] = 4
    with pytest.raises(RuntimeError, match="timed out"):
        ap.check("cuda")
    word.zero_()
    ap.check(ins[0].device)


def test_other_device():
    from tidegs_b200 import appearance as ap

    if torch.cuda.device_count() < 2:
        pytest.skip("one device")
    x = _rand(_gen(0), 50, 16)
    assert torch.equal(ap.layer_norm(x.to("cuda:1")).cpu(), ap.layer_norm(x).cpu())


def test_appearance_colors_into_the_render_path():
    """Features -> norm -> block -> dropout -> SH coefficients -> colors, with
    gradients for the features, the parameters and the base coefficients,
    against the 64-bit oracle chain. The tolerance is the render tests': 1e-4
    of the largest magnitude for values, 1e-3 for gradients (32-bit
    arithmetic and the SH kernels' fast math)."""
    from oracle import render as orr
    from tidegs_b200 import appearance as ap
    from tidegs_b200.render import spherical_harmonics

    n, d, h, deg = 700, 32, 64, 3
    g = _gen(12)
    base = _rand(g, n, 16, 3, scale=0.3)
    feats = _rand(g, n, d)
    nw, nb = 1 + _rand(g, d, scale=0.1), _rand(g, d, scale=0.1)
    ws = (_rand(g, h, d, scale=d ** -0.5), _rand(g, h, d, scale=d ** -0.5), _rand(g, 48, h, scale=h ** -0.5))
    dirs = _rand(g, n, 3)
    ids = torch.arange(n, device="cuda") * 5 + 3
    v = _rand(g, n, 3)
    leaves = [t.requires_grad_(True) for t in (base, feats, nw, nb, *ws)]
    sh = ap.appearance_colors(base, feats, (nw, nb), ws, p=0.2, seed=9, offset=4, ids=ids)
    assert sh.shape == base.shape
    colors = spherical_harmonics(deg, dirs, sh)
    grads = torch.autograd.grad(colors, leaves, v)
    deep = [t.detach().double().cpu().requires_grad_(True) for t in leaves]
    keep = torch.from_numpy(orc.dropout_keep(n, 48, 0.2, 9, 4, ids.cpu().numpy()))
    y = orc.gated_feed_forward(orc.layer_norm(deep[1], deep[2], deep[3]), *deep[4:])
    want = orr.sh_colors(deg, dirs.double().cpu(), deep[0] + (y * keep / 0.8).reshape(n, 16, 3))
    deep_grads = torch.autograd.grad(want, deep, v.double().cpu())
    scale = float(want.detach().abs().max())
    assert float((colors.double().cpu() - want).abs().max()) <= 1e-4 * scale
    for a, e in zip(grads, deep_grads):
        assert float((a.double().cpu() - e).abs().max()) <= 1e-3 * float(e.abs().max())
    # base in 32 bits with a bfloat16 head: base's type and gradient
    half = [t.detach().bfloat16() for t in (feats, nw, nb, *ws)]
    sh = ap.appearance_colors(base, half[0], (half[1], half[2]), tuple(half[3:]))
    assert sh.dtype == torch.float32
    assert torch.equal(torch.autograd.grad(sh, base, torch.ones_like(sh))[0], torch.ones_like(base))
