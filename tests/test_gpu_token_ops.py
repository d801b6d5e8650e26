"""GPU: the token operators (yolopoint_amd/utils/token_ops.py, csrc/token.hip) against their definitions in 64 bits (oracle/token_oracle.py).

Tolerances.  A result of type t is off by half a step of its own value (finfo(t).eps / 2) plus what the fp32 arithmetic in front of that rounding is
off: a small multiple of 2^-24 times the sum of the magnitudes that enter the value.  F32 below is that multiple: the longest chain of roundings
(16 additions in a thread, 10 over the threads of a row, some 10 operations a value) stays under it."""
import ctypes as C
import math

import pytest
import torch

from oracle import token_oracle as O
from yolopoint_amd import _hip
from yolopoint_amd.utils import token_ops as ops

pytestmark = pytest.mark.gpu

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
F32 = 48 * 2.0 ** -24


def near(got, want, magnitude, extra=0.0):
    """|got - want| <= half a step of got's type at the value + F32 * magnitude (+ extra); got on the GPU, want / magnitude in 64 bits."""
    got64 = got.detach().cpu().double()
    inner = F32 * magnitude + extra
    tiny = torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps
    bound = (want.abs() + inner) * torch.finfo(got.dtype).eps / 2 + inner + tiny
    off = (got64 - want).abs()
    assert got.shape == want.shape
    assert bool(torch.isfinite(got64).all())
    assert bool((off <= bound).all()), (float((off / bound).max()), int((off > bound).sum()), got.shape, got.dtype)


def make(cuda, shape, dtype, seed, mean=0.4, std=1.3):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * std + mean).to(dtype).to(cuda)


def norm_forward_bound(x, w, b, eps):
    y, mean, rstd, xhat = O.layer_norm(x, w, b, eps)
    w = 1.0 if w is None else w.double()
    # xhat's own error: the mean's (of the size of the row's values) times rstd, and that of rstd (relative)
    size = (x.double().abs().mean(-1, keepdim=True) + x.double().abs()) * rstd + xhat.abs()
    return y, size * abs(w) + (0.0 if b is None else b.double().abs())


def norm_backward_bound(x, w, dy, eps):
    _, _, rstd, xhat = O.layer_norm(x, None, None, eps)
    dx, dw, db = O.layer_norm_backward(x, w, dy, eps)
    h = dy.double() * (1.0 if w is None else w.double())
    shift = x.double().abs().mean(-1, keepdim=True) * rstd                       # what the rounding of the mean moves xhat by, over 2^-24
    m1, m2 = h.abs().mean(-1, keepdim=True), (h * xhat).abs().mean(-1, keepdim=True)
    dx_size = rstd * (h.abs() + m1 + (xhat.abs() + shift) * (m2 + shift * m1))
    D = x.shape[-1]
    terms = (dy.double().abs() * (xhat.abs() + shift)).reshape(-1, D).sum(0)
    return (dx, dx_size), (dw, 2 * terms), (db, 2 * dy.double().abs().reshape(-1, D).sum(0))   # (twice: up to 96 additions one after the other)


WIDTHS = [1, 2, 3, 4, 5, 7, 8, 9, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 200, 255, 256, 257, 511, 512, 513, 777, 1000, 1023, 1024, 1025, 2047, 2048,
          2049, 4095, 4096, 4097, 8192, 8193, 12345, 16383, 16384]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", WIDTHS)
def test_layer_norm_widths(cuda, D, dtype):
    """Every row shape, from both sides of its border, forward and backward; weights in fp32 or the rows' type."""
    dt = TYPES[dtype]
    rows = 5 if D > 2048 else 67
    wt = torch.float32 if D % 2 else dt
    x, dy = make(cuda, (rows, D), dt, D), make(cuda, (rows, D), dt, D + 1, 0.1, 0.7)
    w, b = make(cuda, (D,), wt, D + 2, 1.0, 0.3), make(cuda, (D,), wt, D + 3, 0.0, 0.5)
    x, w, b = (t.requires_grad_() for t in (x, w, b))
    y = ops.layer_norm(x, w, b, 1e-5)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    xc, wc, bc, dyc = (t.detach().cpu() for t in (x, w, b, dy))
    near(y, *norm_forward_bound(xc, wc, bc, 1e-5))
    for got, (want, size) in zip((dx, dw, db), norm_backward_bound(xc, wc, dyc, 1e-5)):
        near(got, want, size)
    with torch.no_grad():
        assert torch.equal(ops.layer_norm(x, w, b, 1e-5), y)                     # the pass without statistics: the same kernel


@pytest.mark.parametrize("rows", [0, 1, 2, 3, 63, 64, 65, 1000, 5001, 40000])
def test_layer_norm_rows(cuda, rows):
    x, dy = make(cuda, (rows, 72), torch.bfloat16, rows).requires_grad_(), make(cuda, (rows, 72), torch.bfloat16, rows + 1)
    w, b = make(cuda, (72,), torch.float32, 1).requires_grad_(), make(cuda, (72,), torch.float32, 2).requires_grad_()
    y = ops.layer_norm(x, w, b)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    if rows == 0:
        assert y.shape == (0, 72) and dx.shape == (0, 72) and not dw.any() and not db.any()
        return
    near(y, *norm_forward_bound(x.detach().cpu(), w.detach().cpu(), b.detach().cpu(), 1e-5))
    for got, (want, size) in zip((dx, dw, db), norm_backward_bound(x.detach().cpu(), w.detach().cpu(), dy.cpu(), 1e-5)):
        near(got, want, size)
    again = torch.autograd.grad(ops.layer_norm(x, w, b), (x, w, b), dy)
    assert all(torch.equal(p, q) for p, q in zip((dx, dw, db), again))           # no order to depend on


@pytest.mark.parametrize("weight,bias", [(False, False), (True, False), (False, True)])
@pytest.mark.parametrize("dtype", TYPES)
def test_layer_norm_without_weights(cuda, weight, bias, dtype):
    dt = TYPES[dtype]
    x, dy = make(cuda, (33, 100), dt, 5).requires_grad_(), make(cuda, (33, 100), dt, 6)
    w = make(cuda, (100,), torch.float32, 7).requires_grad_() if weight else None
    b = make(cuda, (100,), torch.float32, 8).requires_grad_() if bias else None
    y = ops.layer_norm(x, w, b, eps=1e-3)
    leaves = [t for t in (x, w, b) if t is not None]
    got = torch.autograd.grad(y, leaves, dy)
    cw, cb = None if w is None else w.detach().cpu(), None if b is None else b.detach().cpu()
    near(y, *norm_forward_bound(x.detach().cpu(), cw, cb, 1e-3))
    want = norm_backward_bound(x.detach().cpu(), cw, dy.cpu(), 1e-3)
    near(got[0], *want[0])
    if weight:
        near(got[1], *want[1])
    if bias:
        near(got[-1], *want[2])


def test_layer_norm_frozen_leaves(cuda):
    """Only what needs a gradient gets one: frozen weights, or a frozen input under trained weights."""
    x, dy = make(cuda, (9, 40), torch.float32, 1), make(cuda, (9, 40), torch.float32, 2)
    w, b = make(cuda, (40,), torch.float32, 3), make(cuda, (40,), torch.float32, 4)
    full = torch.autograd.grad(ops.layer_norm(x.requires_grad_(), w.requires_grad_(), b.requires_grad_()), (x, w, b), dy)
    for keep in range(3):
        leaves = [t.detach().requires_grad_(i == keep) for i, t in enumerate((x, w, b))]
        assert torch.equal(torch.autograd.grad(ops.layer_norm(*leaves), leaves[keep], dy)[0], full[keep])


@pytest.mark.parametrize("dtype", TYPES)
def test_layer_norm_reads_slices_and_orders(cuda, dtype):
    """Rows inside wider rows (any first element), one row for all, transposed and channels-first tensors, a gradient that is one value for all."""
    dt = TYPES[dtype]
    base = make(cuda, (6, 10, 131), dt, 9)
    w, b = make(cuda, (50,), torch.float32, 1), make(cuda, (50,), torch.float32, 2)
    for x in (base[..., 1:51], base[..., 7:57], base[:, :1, 3:53], base[:, 2:7, :50], base[1:2, :, 5:55].transpose(0, 1), base[0, 0, 2:52].expand(7, 50),
              base.transpose(1, 2)[:, :50].transpose(1, 2)[..., :10].repeat(1, 1, 5), base[0, 0, 4:54]):
        assert x.shape[-1] == 50
        leaf = x.detach().clone().requires_grad_()
        y = ops.layer_norm(x, w, b)
        assert torch.equal(y, ops.layer_norm(leaf, w, b)) and y.is_contiguous()
        y2 = ops.layer_norm(x.detach().requires_grad_(), w, b)
        assert torch.equal(y, y2)
        v = x.detach().requires_grad_()
        g1, = torch.autograd.grad(ops.layer_norm(v, w, b).sum(), v)               # (an expanded gradient: stride 0)
        g2, = torch.autograd.grad(ops.layer_norm(leaf, w, b), leaf, torch.ones_like(leaf))
        assert torch.equal(g1, g2)
        d = make(cuda, (*x.shape[:-1], 64), dt, 3)[..., 9:59]                     # a gradient inside wider rows
        g1, = torch.autograd.grad(ops.layer_norm(v, w, b), v, d)
        g2, = torch.autograd.grad(ops.layer_norm(leaf, w, b), leaf, d.contiguous())
        assert torch.equal(g1, g2)
    nhwc = make(cuda, (2, 48, 5, 7), dt, 4).to(memory_format=torch.channels_last).permute(0, 2, 3, 1)
    assert torch.equal(ops.layer_norm(nhwc), ops.layer_norm(nhwc.contiguous()))
    wide = make(cuda, (100,), torch.float32, 5)
    assert torch.equal(ops.layer_norm(base[..., :50], wide[::2], wide[1::2]), ops.layer_norm(base[..., :50], wide[::2].contiguous(), wide[1::2].contiguous()))


def test_layer_norm_hard_rows(cuda):
    """Constant rows, rows far from zero, infinities and NaN: what the formula gives, and nothing in the neighbours."""
    x = make(cuda, (8, 300), torch.float32, 1, 0.0, 1.0)
    x[1] = 7.25
    x[2] = 0.0
    x[3] += 4096.0
    clean = ops.layer_norm(x, eps=1e-5)
    assert not clean[1].any() and not clean[2].any()
    near(clean, *norm_forward_bound(x.cpu(), None, None, 1e-5))
    y = x.clone()
    y[4, 17], y[5, 0], y[6, 299] = float("inf"), float("nan"), float("-inf")
    got = ops.layer_norm(y, eps=1e-5)
    assert bool(got[4:7].isnan().all()) and torch.equal(got[[0, 1, 2, 3, 7]], clean[[0, 1, 2, 3, 7]])
    assert bool(ops.layer_norm(torch.zeros(2, 5, device=cuda), eps=0.0).isnan().all())     # 0 / 0


@pytest.mark.parametrize("dtype", TYPES)
def test_layer_norm_far_from_zero(cuda, dtype):
    """Rows whose deviation is one step of their type: the rounding of the mean must not show.  (x - mean) is exact, the mean's rounding is taken off, so
    y is off by a few 2^-24 of itself in fp32 and f16; bf16: by the mean's rounding, 4 * 2^-24 of 2^8 deviations."""
    dt = TYPES[dtype]
    step = torch.finfo(dt).eps * 1024.0
    g = torch.Generator().manual_seed(1)
    for D in (64, 777, 5000):
        x = (1024.0 + step * torch.randint(0, 3, (9, D), generator=g).double()).to(dt)
        y, _, rstd, xhat = O.layer_norm(x, None, None, 0.0 if dtype == "f32" else 1e-9)
        got = ops.layer_norm(x.to(cuda), eps=0.0 if dtype == "f32" else 1e-9)
        near(got, y, xhat.abs() + 1.0, 4 * 2.0 ** -24 * 1024.0 * float(rstd.max()) if dtype == "bf16" else 0.0)


def test_layer_norm_large_strides(cuda):
    """Rows more than 2^31 elements into a tensor."""
    base = torch.zeros((1 << 31) + 4096, dtype=torch.bfloat16, device=cuda)
    x = base.as_strided((3, 64), (1 << 30, 1), 1027)
    x.copy_(make(cuda, (3, 64), torch.bfloat16, 3))
    assert torch.equal(ops.layer_norm(x), ops.layer_norm(x.contiguous()))
    leaf = x.detach().requires_grad_()
    dy = make(cuda, (3, 64), torch.bfloat16, 4)
    dense = x.contiguous().requires_grad_()
    assert torch.equal(torch.autograd.grad(ops.layer_norm(leaf), leaf, dy)[0], torch.autograd.grad(ops.layer_norm(dense), dense, dy)[0])


# ------------------------------------------------------------------------------------------------------------------ dropout
SIZES = [1, 2, 3, 4, 5, 7, 8, 9, 11, 15, 16, 17, 63, 64, 65, 1000, 4099, 100003]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", SIZES)
def test_dropout_mask_and_values(cuda, n, dtype):
    dt = TYPES[dtype]
    x, r, dy = (make(cuda, (n,), dt, n + i) for i in range(3))
    x[x == 0] = 1.0
    for p, seed, offset in ((0.1, 1, 0), (0.5, (1 << 64) - 1, 3), (0.93, 12345678901234567890, (1 << 63) + 5)):
        keep = O.keep_mask(n, p, seed, offset)
        y = ops.dropout(x, p, (seed, offset))
        assert torch.equal(y.cpu() != 0, keep)
        near(y, O.dropout(x.cpu(), p, seed, offset), 0.0, 2.0 ** -24 * x.cpu().double().abs() / (1 - p))
        z = ops.dropout(x, p, (seed, offset), residual=r)
        want = O.dropout(x.cpu(), p, seed, offset, r.cpu())
        near(z, want, 0.0, 2.0 ** -24 * want.abs())
        if dt != torch.float32:                                                    # (the fp32 sum's nearest value: how torch converts 64 bits too)
            assert torch.equal(z.cpu(), want.to(dt)) and torch.equal(z.cpu(), want.float().to(dt))
        a, c = x.clone().requires_grad_(), r.clone().requires_grad_()
        da, dc = torch.autograd.grad(ops.dropout(a, p, (seed, offset), residual=c), (a, c), dy)
        assert torch.equal(da, ops.dropout(dy, p, (seed, offset))) and torch.equal(dc, dy)
        da, = torch.autograd.grad(ops.dropout(a, p, (seed, offset)), a, dy)
        assert torch.equal(da, ops.dropout(dy, p, (seed, offset)))


def test_dropout_rates_at_their_ends(cuda):
    x = make(cuda, (4099,), torch.bfloat16, 1)
    r = make(cuda, (4099,), torch.bfloat16, 2)
    assert torch.equal(ops.dropout(x, 0.0, None), x) and torch.equal(ops.dropout(x, 1e-6, (1, 2)), x)
    assert not ops.dropout(x, 1.0, (1, 2)).any() and torch.equal(ops.dropout(x, 1.0, (1, 2), residual=r), r)
    assert torch.equal(ops.dropout(x, 0.0, (1, 2), residual=r), (x.float() + r.float()).bfloat16())
    bad = torch.full((4099,), float("nan"), device=cuda, dtype=torch.bfloat16)
    bad[::3] = float("inf")
    keep = O.keep_mask(4099, 0.4, 3, 4)
    got = ops.dropout(bad, 0.4, (3, 4)).cpu()
    assert not got[~keep].any() and bool((~got[keep].isfinite()).all())            # dropped means 0, whatever it held
    got = ops.dropout(bad, 0.4, (3, 4), residual=r).cpu()
    assert torch.equal(got[~keep], r.cpu()[~keep])
    assert ops.dropout(x[:0], 0.5, (1, 2)).numel() == 0


def test_dropout_does_not_depend_on_shape_order_or_place(cuda):
    x = make(cuda, (4, 6, 50), torch.float16, 1)
    x[x == 0] = 1.0
    y = ops.dropout(x, 0.3, (8, 9))
    assert torch.equal(y.view(-1), ops.dropout(x.view(-1), 0.3, (8, 9))) and torch.equal(y, ops.dropout(x.transpose(0, 1).contiguous().transpose(0, 1), 0.3, (8, 9)))
    big = torch.zeros(1201, device=cuda, dtype=torch.float16)
    big[1:] = x.view(-1)
    assert torch.equal(ops.dropout(big[1:], 0.3, (8, 9)), y.view(-1))               # two bytes past a border
    one = x[:1, :1].expand(4, 6, 50)
    assert torch.equal(ops.dropout(one, 0.3, (8, 9)), ops.dropout(one.contiguous(), 0.3, (8, 9)))


def test_dropout_state_on_the_device(cuda):
    x = make(cuda, (1000,), torch.bfloat16, 1)
    state = torch.tensor([77, 5], device=cuda)
    assert torch.equal(ops.dropout(x, 0.25, state), ops.dropout(x, 0.25, (77, 5)))
    state[0] = -3                                                                  # (the 64 bits of 2^64 - 3)
    assert torch.equal(ops.dropout(x, 0.25, state), ops.dropout(x, 0.25, ((1 << 64) - 3, 5)))
    leaf = x.clone().requires_grad_()
    y = ops.dropout(leaf, 0.25, state)
    state[1] += 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):    # another mask than the forward pass's: refused
        torch.autograd.grad(y, leaf, x)


def test_dropout_past_32_bits(cuda):
    """Elements behind 2^32, in the mask and in the addresses."""
    n = (1 << 32) + 77
    x = torch.ones(n, dtype=torch.bfloat16, device=cuda)
    y = ops.dropout(x, 0.5, (4, 2))
    for start in (0, (1 << 31) - 40, (1 << 32) - 40, n - 70):
        assert torch.equal(y[start:start + 70].cpu() != 0, O.keep_mask(70, 0.5, 4, 2, start=start))


# ------------------------------------------------------------------------------------------------------------------ the fused operator
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [1, 3, 4, 7, 8, 12, 33, 64, 100, 256, 257, 511, 1000, 1024, 2050, 4100, 9000, 16384])
def test_fused_equals_its_parts_and_the_formula(cuda, D, dtype):
    dt = TYPES[dtype]
    rows = 3 if D > 4096 else 37
    wt = torch.float32 if D % 2 == 0 else dt
    for p in (0.0, 0.2):
        x, r, dy, dz = (make(cuda, (rows, D), dt, D + i) for i in range(4))
        w, b = make(cuda, (D,), wt, D + 4, 1.0, 0.3), make(cuda, (D,), wt, D + 5)
        leaves = [t.requires_grad_() for t in (x, r, w, b)]
        rng = (99, D)
        y, z = ops.dropout_add_layer_norm(x, r, w, b, p=p, rng=rng)
        assert torch.equal(z, ops.dropout(x, p, rng, residual=r)) and torch.equal(y, ops.layer_norm(z.detach(), w, b))
        xc, rc, wc, bc, dyc, dzc = (t.detach().cpu() for t in (x, r, w, b, dy, dz))
        zc = O.stored_sum(xc, rc, p, *rng)
        if dt != torch.float32:
            assert torch.equal(z.detach().cpu(), zc)
        zc = z.detach().cpu()                                                     # (fp32: the sum as stored, a step from the oracle's at most)
        near(y, *norm_forward_bound(zc, wc, bc, 1e-5))
        got = torch.autograd.grad((y, z), leaves, (dy, dz), retain_graph=True)
        again = torch.autograd.grad((y, z), leaves, (dy, dz), retain_graph=True)
        assert all(torch.equal(i, j) for i, j in zip(got, again))
        (dr, dr_size), dw, db = norm_backward_bound(zc, wc, dyc, 1e-5)
        dr, dr_size = dr + dzc.double(), dr_size + dzc.double().abs()
        keep = (O.keep_mask(rows * D, p, *rng).view(rows, D) if p else torch.ones(rows, D)).double() * O.drop_scale(p)
        near(got[0], dr * keep, dr_size * keep)
        near(got[1], dr, dr_size)
        near(got[2], *dw)
        near(got[3], *db)
        assert p == 0.0 or not got[0].cpu()[keep == 0].any()
        # the gradient of one result alone
        only_y = torch.autograd.grad(y, leaves, dy, retain_graph=True)
        near(only_y[0], (dr - dzc.double()) * keep, dr_size * keep)
        assert torch.equal(only_y[2], got[2]) and torch.equal(only_y[3], got[3])
        only_z = torch.autograd.grad(z, leaves, dz, retain_graph=True)
        assert torch.equal(only_z[1], dz) and torch.equal(only_z[0], ops.dropout(dz, p, rng)) and not only_z[2].any() and not only_z[3].any()
        with torch.no_grad():
            y2, z2 = ops.dropout_add_layer_norm(x, r, w, b, p=p, rng=rng)
        assert torch.equal(y, y2) and torch.equal(z, z2)


def test_fused_of_a_tensor_with_itself_and_dropped_whole(cuda):
    """x and residual the same leaf: its gradient is the sum of both.  p = 1: the residual's norm, no gradient through the branch."""
    x, dy, dz = (make(cuda, (21, 88), torch.float32, i) for i in range(3))
    a, b = x.clone().requires_grad_(), x.clone().requires_grad_()
    for p in (0.0, 0.4):
        one = torch.autograd.grad(ops.dropout_add_layer_norm(a, a, p=p, rng=(1, 2)), a, (dy, dz))[0]
        two = torch.autograd.grad(ops.dropout_add_layer_norm(a, b, p=p, rng=(1, 2)), (a, b), (dy, dz))
        assert torch.equal(one, two[0] + two[1])
    y, z = ops.dropout_add_layer_norm(a, b, p=1.0, rng=(1, 2))
    assert torch.equal(z, b) and torch.equal(y, ops.layer_norm(b))
    da, db = torch.autograd.grad((y, z), (a, b), (dy, dz))
    assert not da.any() and bool(db.any())


def test_fused_many_rows(cuda):
    """More rows than workgroups: every workgroup walks, the partial sums of all of them join."""
    rows, D, p, rng = 30011, 136, 0.1, (3, 1)
    x, r, dy, dz = (make(cuda, (rows, D), torch.bfloat16, i) for i in range(4))
    w, b = make(cuda, (D,), torch.float32, 5).requires_grad_(), make(cuda, (D,), torch.float32, 6).requires_grad_()
    x.requires_grad_(), r.requires_grad_()
    y, z = ops.dropout_add_layer_norm(x, r, w, b, p=p, rng=rng)
    assert torch.equal(z.detach().cpu(), O.stored_sum(x.detach().cpu(), r.detach().cpu(), p, *rng))
    got = torch.autograd.grad((y, z), (x, r, w, b), (dy, dz))
    (dr, size), dw, db = norm_backward_bound(z.detach().cpu(), w.detach().cpu(), dy.cpu(), 1e-5)
    near(got[1], dr + dz.cpu().double(), size + dz.cpu().double().abs())
    near(got[2], *dw)
    near(got[3], *db)


def test_results_stay_inside_their_buffers(cuda):
    """The C entry points on buffers inside larger ones: the bytes before and behind each result stay as they were."""
    l = _hip.lib()
    for rows, D, dt in ((5, 61, torch.bfloat16), (3, 7, torch.float16), (4, 130, torch.float32), (2, 1, torch.float16), (6, 1001, torch.bfloat16)):
        n, pad = rows * D, 64
        x, r = make(cuda, (rows, D), dt, 1), make(cuda, (rows, D), dt, 2)
        mark = 3.0

        def room(m, t=dt):
            return torch.full((m + 2 * pad,), mark, dtype=t, device=cuda)

        def inner(t):
            return t.data_ptr() + pad * t.element_size()

        y, z, mean, rstd = room(n), room(n), room(rows, torch.float32), room(rows, torch.float32)
        how = dict(rows=rows, D=D, dtype=_hip.dtype_code(dt), wdtype=_hip.YP_F32, eps=1e-5, p=0.25, seed=1, offset=2, x_stride=D)
        _hip.check(l.yp_layer_norm_fwd(C.byref(_hip.YpLayerNormDesc(x=x.data_ptr(), res=r.data_ptr(), res_stride=D, z=inner(z), y=inner(y), mean=inner(mean), rstd=inner(rstd), **how)),
                                       _hip.stream_ptr()))
        dres, dx, dw, db = room(n), room(n), room(D, torch.float32), room(D, torch.float32)
        nb = l.yp_layer_norm_bwd_workspace_bytes(rows, D, _hip.dtype_code(dt))
        ws = torch.full((nb // 4 + 2 * pad,), mark, device=cuda)
        _hip.check(l.yp_layer_norm_bwd(C.byref(_hip.YpLayerNormDesc(x=inner(z), dy=x.data_ptr(), dz=r.data_ptr(), dy_stride=D, dz_stride=D, mean=inner(mean), rstd=inner(rstd), dres=inner(dres),
                                                                    dx=inner(dx), dweight=inner(dw), dbias=inner(db), workspace=inner(ws), workspace_bytes=nb, **how)), _hip.stream_ptr()))
        d = room(n)
        _hip.check(l.yp_dropout(x.data_ptr(), r.data_ptr(), inner(d), n, _hip.dtype_code(dt), 0.25, 1, 2, None, _hip.stream_ptr()))
        assert torch.equal(d[pad:pad + n], z[pad:pad + n])
        for t in (y, z, mean, rstd, dres, dx, dw, db, ws, d):
            assert bool((t[:pad] == mark).all()) and bool((t[-pad:] == mark).all())


# ------------------------------------------------------------------------------------------------------------------ rotary positions
def rotary_case(cuda, B, T, Hq, Hk, D, R, dtype, layout, interleaved, axes, kind, seed=0):
    dt = TYPES[dtype]
    g = torch.Generator().manual_seed(seed + D + T)
    inv, scale = ops.rotary_frequencies(R, 1000.0, axes=axes)
    if kind == "f32":
        pos = torch.rand((B, T, axes) if axes == 2 else (B, T), generator=g) * 900 - 100
    else:
        pos = torch.randint(-50, 5000, (B, T, axes) if axes == 2 else (B, T), generator=g, dtype=torch.int64).to(torch.int32 if kind == "i32" else torch.int64)
    shape = (lambda h: (B, T, h, D)) if layout == "bthd" else (lambda h: (B, h, T, D))
    return make(cuda, shape(Hq), dt, seed), make(cuda, shape(Hk), dt, seed + 1) if Hk else None, pos, inv, scale


def near_rotary(got, x, pos, inv, interleaved, layout, scale, inverse=False):
    """A turned pair is off by the rounding of its angle's cosine and sine (under 4 * 2^-24 of the pair's length) and half a step."""
    want = O.rotary(x.detach().cpu(), pos, inv, interleaved, layout, scale, inverse)
    half = inv.numel()
    size = x.detach().cpu().double().abs()
    a, b = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved else (slice(0, half), slice(half, 2 * half))
    length = torch.zeros_like(size)
    length[..., a] = length[..., b] = size[..., a] + size[..., b]
    near(got, want, 0.0, 8 * 2.0 ** -24 * scale * length)
    assert torch.equal(got[..., 2 * half:].cpu(), x[..., 2 * half:].detach().cpu())


@pytest.mark.parametrize("layout", ["bthd", "bhtd"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D,R,axes", [(2, 2, 1), (4, 4, 2), (6, 2, 1), (10, 6, 1), (16, 16, 1), (20, 12, 2), (64, 64, 1), (64, 32, 2), (80, 40, 1), (96, 96, 2), (128, 128, 1),
                                      (128, 64, 2), (130, 66, 1), (256, 256, 1), (1024, 1024, 2), (1024, 2, 1)])
def test_rotary_forms(cuda, D, R, axes, dtype, interleaved, layout):
    for B, T, Hq, Hk, kind in ((2, 7, 4, 2, "i64"), (3, 1, 5, 0, "f32"), (1, 33, 1, 3, "i32")):
        q, k, pos, inv, _ = rotary_case(cuda, B, T, Hq, Hk, D, R, dtype, layout, interleaved, axes, kind)
        scale = 1.0 if Hk else 1.2
        q.requires_grad_()
        dq = make(cuda, q.shape, q.dtype, 7)
        if k is None:
            out = ops.rotary(q, pos.to(cuda), inv.to(cuda), interleaved=interleaved, layout=layout, scale=scale)
            near_rotary(out, q, pos, inv, interleaved, layout, scale)
            gq, = torch.autograd.grad(out, q, dq)
        else:
            k.requires_grad_()
            dk = make(cuda, k.shape, k.dtype, 8)
            out, ko = ops.rotary(q, pos.to(cuda), inv.to(cuda), k=k, interleaved=interleaved, layout=layout, scale=scale)
            near_rotary(out, q, pos, inv, interleaved, layout, scale)
            near_rotary(ko, k, pos, inv, interleaved, layout, scale)
            gq, gk = torch.autograd.grad((out, ko), (q, k), (dq, dk), retain_graph=True)
            near_rotary(gk, dk, pos, inv, interleaved, layout, scale, True)
            only, = torch.autograd.grad(ko, k, dk, retain_graph=True)                # one of the two results is used
            assert torch.equal(only, gk)
            with torch.no_grad():                                                    # each alone: the same bits
                assert torch.equal(ops.rotary(k, pos.to(cuda), inv.to(cuda), interleaved=interleaved, layout=layout, scale=scale), ko)
        near_rotary(gq, dq, pos, inv, interleaved, layout, scale, True)
        with torch.no_grad():
            a = q.detach().clone()
            b = None if k is None else k.detach().clone()
            back = ops.rotary(a, pos.to(cuda), inv.to(cuda), k=b, interleaved=interleaved, layout=layout, scale=scale, inplace=True)
            assert (back if k is None else back[0]) is a and torch.equal(a, out) and (k is None or torch.equal(b, ko))


def test_rotary_many_tokens_and_heads(cuda):
    """More tokens than workgroups hold at once, heads that do not divide among the threads."""
    for B, T, Hq, Hk, D in ((5, 3001, 7, 2, 64), (1, 1, 130, 3, 128), (40, 700, 3, 3, 32), (2, 9000, 17, 0, 128)):
        q, k, pos, inv, scale = rotary_case(cuda, B, T, Hq, Hk, D, D, "bf16", "bthd", False, 1, "i64")
        out = ops.rotary(q, pos.to(cuda), inv.to(cuda), k=k)
        near_rotary(out if k is None else out[0], q, pos, inv, False, "bthd", 1.0)
        if k is not None:
            near_rotary(out[1], k, pos, inv, False, "bthd", 1.0)


def test_rotary_reads_slices_of_a_joint_projection(cuda):
    B, T, H, D = 2, 11, 4, 48
    joint = make(cuda, (B, T, 3 * H * D + 5), torch.bfloat16, 1)
    parts = joint.as_strided((B, T, 3, H, D), (joint.stride(0), joint.stride(1), H * D, D, 1), 3)
    q, k = parts[:, :, 0], parts[:, :, 1]
    inv = ops.rotary_frequencies(32)[0].to(cuda)
    pos = torch.arange(T, device=cuda)
    a, b = ops.rotary(q, pos, inv, k=k)
    c, d = ops.rotary(q.contiguous(), pos, inv, k=k.contiguous())
    assert torch.equal(a, c) and torch.equal(b, d) and a.is_contiguous()
    e, f = ops.rotary(q.transpose(1, 2), pos, inv, k=k.transpose(1, 2), layout="bhtd")
    assert torch.equal(e.transpose(1, 2), c) and torch.equal(f.transpose(1, 2), d)
    before = joint.clone()
    ops.rotary(q, pos, inv, k=k, inplace=True)
    assert torch.equal(q, c) and torch.equal(k, d)
    before.as_strided(parts.shape, parts.stride(), 3)[:, :, :2] = parts[:, :, :2]
    assert torch.equal(before, joint)                                              # nothing but q and k was written
    odd = make(cuda, (B, T, H, 2 * D), torch.bfloat16, 2)[..., ::2]
    assert torch.equal(ops.rotary(odd, pos, inv), ops.rotary(odd.contiguous(), pos, inv))
    for a, b in ((odd, None), (q[:, :, :1].expand(B, T, H, D), None), (q, q), (q, q[:, :, 1:]), (q[:, :-1], joint.as_strided((B, T - 1, H, D), q.stride(), 3 + 3 * H * D)),
                 (q, joint.as_strided((B, T, H, D), (q.stride(0), q.stride(1), D, 1), 3 + D // 2)), (q[:, :-1], joint.as_strided((B, T - 1, 3 * H, D), (q.stride(0), q.stride(1), D, 1), 3 + H * D))):
        with pytest.raises(_hip.YpError):                                          # an element twice
            ops.rotary(a, pos[:a.shape[1]], inv, k=b, inplace=True)
    heads = make(cuda, (B, 3, H, T, D), torch.bfloat16, 4)                         # joint per batch entry, heads in front
    want = ops.rotary(heads[:, 0], pos, inv, k=heads[:, 2], layout="bhtd")
    ops.rotary(heads[:, 0], pos, inv, k=heads[:, 2], layout="bhtd", inplace=True)
    assert torch.equal(heads[:, 0], want[0]) and torch.equal(heads[:, 2], want[1])
    leaf = q.detach().clone().requires_grad_()
    h = leaf * 1.0
    y = h * h
    with torch.no_grad():
        ops.rotary(h, pos, inv, inplace=True)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):    # autograd sees the write
        y.sum().backward()


def test_rotary_positions(cuda):
    """Every way to say the same positions; far ones; the limits of 32 bits."""
    B, T = 3, 9
    q = make(cuda, (B, T, 2, 64), torch.float32, 1)
    inv = ops.rotary_frequencies(64)[0].to(cuda)
    at = torch.arange(T, device=cuda) + 1000
    want = ops.rotary(q, at, inv)
    for pos in (1000, at.int(), at.float(), at[None], at.expand(B, T), at.repeat(B, 1), torch.stack([at, at], 1)[:, 0], at.repeat_interleave(2)[::2]):
        assert torch.equal(ops.rotary(q, pos, inv), want)
    each = torch.tensor([[5], [0], [70000]], device=cuda) + torch.arange(T, device=cuda)
    got = ops.rotary(q, each, inv)
    for b in range(B):
        assert torch.equal(got[b:b + 1], ops.rotary(q[b:b + 1], int(each[b, 0]), inv))
    two = torch.rand(B, T, 2, device=cuda) * 640
    assert torch.equal(ops.rotary(q, two[:1], inv), ops.rotary(q, two[0], inv)) and torch.equal(ops.rotary(q, two[:1].expand(B, T, 2), inv), ops.rotary(q, two[0], inv))
    assert torch.equal(ops.rotary(q, two.transpose(0, 2).contiguous().transpose(0, 2), inv), ops.rotary(q, two, inv))
    for far in (10 ** 6, 2 ** 31 + 3, 2 ** 40, -(2 ** 33)):                          # 64-bit angles: a position p keeps 2^-53 |p| radians, twice rounded
        got, pos = ops.rotary(q, far, inv), (torch.arange(T) + far)
        want = O.rotary(q.cpu(), pos, inv.cpu(), False, "bthd", 1.0)
        pair = (q[..., :32].abs() + q[..., 32:].abs()).repeat(1, 1, 1, 2).cpu().double()
        near(got, want, 0.0, (8 * 2.0 ** -24 + 4 * abs(far) * 2.0 ** -53) * pair)
    still = ops.rotary(q, torch.zeros(T, device=cuda), inv)
    assert torch.equal(still, q)
    bad = at.float()
    bad[2] = float("nan")
    got = ops.rotary(q, bad, inv)
    assert bool(got[:, 2].isnan().all()) and torch.equal(got[:, 3:], ops.rotary(q, at, inv)[:, 3:])


def test_rotary_empty(cuda):
    inv = ops.rotary_frequencies(8)[0].to(cuda)
    for shape in ((0, 4, 2, 8), (2, 0, 2, 8), (2, 4, 0, 8)):
        assert ops.rotary(torch.empty(shape, device=cuda), 0, inv).shape == shape


# ------------------------------------------------------------------------------------------------------------------ refusals
def test_refusals(cuda):
    x, w = torch.randn(4, 8, device=cuda), torch.randn(8, device=cuda)
    inv = ops.rotary_frequencies(8)[0].to(cuda)
    q = torch.randn(2, 5, 3, 8, device=cuda)
    at = torch.arange(5, device=cuda)
    calls = [lambda: ops.layer_norm(x.double()), lambda: ops.layer_norm(x.int()), lambda: ops.layer_norm(x, w[:7]), lambda: ops.layer_norm(x, w.half()),
             lambda: ops.layer_norm(x.half(), w.half(), w), lambda: ops.layer_norm(x, w.cpu()), lambda: ops.layer_norm(x, eps=-1.0), lambda: ops.layer_norm(x, eps=float("nan")),
             lambda: ops.layer_norm(torch.zeros((), device=cuda)), lambda: ops.layer_norm(x[:, :0]), lambda: ops.layer_norm(torch.zeros(1, 16385, device=cuda)),
             lambda: ops.dropout(x, 0.5, None), lambda: ops.dropout(x, -0.1, (1, 2)), lambda: ops.dropout(x, 1.1, (1, 2)), lambda: ops.dropout(x, float("nan"), (1, 2)),
             lambda: ops.dropout(x, 0.5, 7), lambda: ops.dropout(x, 0.5, (1, 2, 3)), lambda: ops.dropout(x, 0.5, (1.5, 2)), lambda: ops.dropout(x, "a", (1, 2)),
             lambda: ops.dropout(x, 0.5, (1 << 64, 0)), lambda: ops.dropout(x, 0.5, (-1, 0)), lambda: ops.dropout(x, 0.5, torch.tensor([1, 2])),
             lambda: ops.dropout(x, 0.5, torch.tensor([1, 2], dtype=torch.int32, device=cuda)), lambda: ops.dropout(x, 0.5, torch.tensor([1, 2, 3], device=cuda)),
             lambda: ops.dropout(x, 0.5, (1, 2), residual=x[:2]), lambda: ops.dropout(x, 0.5, (1, 2), residual=x.half()), lambda: ops.dropout(x, 0.5, (1, 2), residual=x.cpu()),
             lambda: ops.dropout_add_layer_norm(x, x[:1]), lambda: ops.dropout_add_layer_norm(x, x.half()), lambda: ops.dropout_add_layer_norm(x, None),
             lambda: ops.dropout_add_layer_norm(x, x, p=0.5), lambda: ops.dropout_add_layer_norm(x, x, w[:3]),
             lambda: ops.rotary(q[0], at, inv), lambda: ops.rotary(q, at, inv.float()), lambda: ops.rotary(q, at, inv.repeat(2)), lambda: ops.rotary(q, at, inv[:0]),
             lambda: ops.rotary(q, at[:4], inv), lambda: ops.rotary(q, at.double(), inv), lambda: ops.rotary(q, at.cpu(), inv), lambda: ops.rotary(q, at, inv.cpu()),
             lambda: ops.rotary(q, 1.5, inv), lambda: ops.rotary(q, True, inv), lambda: ops.rotary(q, 1 << 63, inv), lambda: ops.rotary(q, at, inv, layout="tbhd"),
             lambda: ops.rotary(q, at, inv, k=q[:1]), lambda: ops.rotary(q, at, inv, k=q[..., :6]), lambda: ops.rotary(q, at, inv, k=q.half()),
             lambda: ops.rotary(q, torch.zeros(5, 2, device=cuda), inv[:3]), lambda: ops.rotary(q, torch.zeros(2, 5, 3, device=cuda), inv),
             lambda: ops.rotary(q.clone().requires_grad_(), at, inv, inplace=True)]
    for i, call in enumerate(calls):
        with pytest.raises(_hip.YpError):
            call()
            print("call", i, "was not refused")


def test_second_differentiation_is_refused(cuda):
    x = torch.randn(4, 8, device=cuda, requires_grad=True)
    inv = ops.rotary_frequencies(8)[0].to(cuda)
    for f in (lambda: ops.layer_norm(x), lambda: ops.dropout(x, 0.5, (1, 2)), lambda: ops.dropout_add_layer_norm(x, x)[0], lambda: ops.rotary(x.view(1, 4, 1, 8), 0, inv)):
        g, = torch.autograd.grad(f().square().sum(), x, create_graph=True)
        with pytest.raises(RuntimeError):
            g.sum().backward()


def test_written_inputs_are_refused_in_the_backward_pass(cuda):
    x = torch.randn(4, 8, device=cuda)
    a = x.clone().requires_grad_()
    h = a * 1.0
    y = ops.layer_norm(h)
    h.mul_(2.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_frequencies_are_a_table(cuda):
    """A table that asks for a gradient would get none: refused."""
    q = torch.randn(2, 5, 3, 8, device=cuda)
    inv = ops.rotary_frequencies(8)[0].to(cuda).requires_grad_()
    for kw in ({}, {"inplace": True}):
        with pytest.raises(_hip.YpError, match="no gradient"):
            ops.rotary(q, 0, inv, **kw)


def test_a_written_state_is_refused_in_the_backward_pass(cuda):
    x = torch.randn(4, 8, device=cuda, requires_grad=True)
    for f in (lambda s: ops.dropout(x, 0.5, s), lambda s: ops.dropout_add_layer_norm(x, x, p=0.5, rng=s)[0]):
        state = torch.tensor([3, 4], device=cuda)
        y = f(state)
        state[1] += 1
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.sum().backward()


def test_a_graph_kept_for_a_second_pass(cuda):
    """retain_graph: the second pass gives the same bits; without it, what was saved is gone."""
    x, w = make(cuda, (37, 100), torch.bfloat16, 1).requires_grad_(), make(cuda, (100,), torch.float32, 2).requires_grad_()
    inv = ops.rotary_frequencies(20)[0].to(cuda)
    at = torch.arange(37, device=cuda)
    y = ops.rotary(ops.dropout_add_layer_norm(ops.layer_norm(x, w), ops.dropout(x, 0.2, (5, 6)), w, p=0.1, rng=(5, 7))[0].view(1, 37, 5, 20), at, inv)
    dy = make(cuda, (1, 37, 5, 20), torch.bfloat16, 3)
    first = torch.autograd.grad(y, (x, w), dy, retain_graph=True)
    second = torch.autograd.grad(y, (x, w), dy)
    assert all(torch.equal(a, b) for a, b in zip(first, second))
    with pytest.raises(RuntimeError, match="second time"):
        torch.autograd.grad(y, (x, w), dy)


def test_inference_mode(cuda):
    """Inference tensors: results as under no_grad; in place too."""
    x, w = make(cuda, (9, 64), torch.float16, 1), make(cuda, (64,), torch.float16, 2).requires_grad_()
    inv = ops.rotary_frequencies(32)[0].to(cuda)
    with torch.no_grad():
        want = ops.dropout_add_layer_norm(x, x, w, p=0.3, rng=(1, 2)), ops.rotary(x.view(1, 9, 2, 32), 7, inv)
    with torch.inference_mode():
        got = ops.dropout_add_layer_norm(x, x, w, p=0.3, rng=(1, 2)), ops.rotary(x.view(1, 9, 2, 32), 7, inv)
        q = x.clone().view(1, 9, 2, 32)
        ops.rotary(q, 7, inv, inplace=True)
        assert torch.equal(q, want[1])
        assert torch.equal(ops.layer_norm(got[0][1], w), want[0][0])
    assert torch.equal(got[0][0], want[0][0]) and torch.equal(got[0][1], want[0][1]) and torch.equal(got[1], want[1])


def test_views_that_are_negated_when_read(cuda):
    """The imaginary part of a conjugate holds its values with the other sign: operands, positions and gradients."""
    c = torch.complex(make(cuda, (50, 1), torch.float32, 1), make(cuda, (50, 1), torch.float32, 2)).conj()
    x, r = c.imag, make(cuda, (50, 1), torch.float32, 3)
    assert x.is_neg()
    dense = x.clone()
    assert not dense.is_neg()
    assert torch.equal(ops.dropout_add_layer_norm(x, r)[1], dense + r) and torch.equal(ops.dropout_add_layer_norm(r, x)[1], dense + r)
    assert torch.equal(ops.dropout(x, 0.5, (1, 2), residual=x), ops.dropout(dense, 0.5, (1, 2), residual=dense))
    w = c[:1, 0].imag
    assert torch.equal(ops.layer_norm(r, None, w), ops.layer_norm(r, None, w.clone()))
    inv = ops.rotary_frequencies(8)[0].to(cuda)
    q = make(cuda, (1, 50, 3, 8), torch.float32, 4)
    assert torch.equal(ops.rotary(q, x[:, 0], inv), ops.rotary(q, dense[:, 0].contiguous(), inv))
    a = r.clone().requires_grad_()
    got, = torch.autograd.grad(ops.dropout_add_layer_norm(a, r, p=0.5, rng=(1, 2)), a, (x, x))
    want, = torch.autograd.grad(ops.dropout_add_layer_norm(a, r, p=0.5, rng=(1, 2)), a, (dense, dense))
    assert torch.equal(got, want)
    view = torch._neg_view(q)
    got = ops.rotary(view, 3, inv)
    assert torch.equal(got, ops.rotary(-q, 3, inv))
    with pytest.raises(_hip.YpError):
        ops.rotary(view, 3, inv, inplace=True)


# ------------------------------------------------------------------------------------------------------------------ streams and graphs
def test_side_stream(cuda):
    """Launches go to the current stream: work queued in front of them on it is seen without a synchronisation."""
    x, r = make(cuda, (4000, 256), torch.bfloat16, 1), make(cuda, (4000, 256), torch.bfloat16, 2)
    want = ops.dropout_add_layer_norm(x * 2, r, p=0.1, rng=(1, 2))
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        slow = x
        for _ in range(50):
            slow = slow * 1.0
        got = ops.dropout_add_layer_norm(slow * 2, r, p=0.1, rng=(1, 2))
    torch.cuda.current_stream().wait_stream(st)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_captured_training_pass_draws_new_masks(cuda):
    """Forward and backward in one graph, the generator's state advanced between replays: every replay equals the eager pass of that state.  Two graphs
    at once share nothing."""
    rows, D = 300, 200
    data = [make(cuda, (rows, D), torch.bfloat16, i) for i in range(4)]
    w0, b0 = make(cuda, (D,), torch.float32, 5), make(cuda, (D,), torch.float32, 6)

    def step(leaves, dy, dz, rng):
        x, r, w, b = leaves
        y, z = ops.dropout_add_layer_norm(x, r, w, b, p=0.2, rng=rng)
        return (y.detach(), z.detach(), *torch.autograd.grad((y, z), leaves, (dy, dz)))

    def captured(state):
        st = torch.cuda.Stream()
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            leaves = [t.clone().requires_grad_() for t in (data[0], data[1], w0, b0)]
            for _ in range(2):
                step(leaves, data[2], data[3], state)
        torch.cuda.current_stream().wait_stream(st)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=st):
            out = step(leaves, data[2], data[3], state)
        return graph, out, leaves
    states = [torch.tensor([11, 0], device=cuda), torch.tensor([12, 40], device=cuda)]
    runs = [captured(s) for s in states]
    for i in range(4):
        for s, (graph, out, _), seed, base in zip(states, runs, (11, 12), (0, 40)):
            graph.replay()
            torch.cuda.synchronize()
            eager = step([t.clone().requires_grad_() for t in (data[0], data[1], w0, b0)], data[2], data[3], (seed, base + i))
            assert all(torch.equal(p, q) for p, q in zip(out, eager)), i
            s[1] += 1
    runs[0][0].replay(), runs[1][0].replay()                                         # back to back
    torch.cuda.synchronize()
    for (_, out, _), seed, base in zip(runs, (11, 12), (4, 44)):
        eager = step([t.clone().requires_grad_() for t in (data[0], data[1], w0, b0)], data[2], data[3], (seed, base))
        assert all(torch.equal(p, q) for p, q in zip(out, eager))


def test_captured_first_call_of_a_wide_norm(cuda):
    """The largest rows, forward and backward captured with no call before: what the launches ask the runtime for may be asked during a capture."""
    D = 16000
    x0, dy, w0 = make(cuda, (7, D), torch.float16, 1), make(cuda, (7, D), torch.float16, 2), make(cuda, (D,), torch.float16, 3)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        x, w = x0.clone().requires_grad_(), w0.clone().requires_grad_()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        y = ops.layer_norm(x, w)
        out = (y.detach(), *torch.autograd.grad(y, (x, w), dy))
    for i in range(3):
        graph.replay()
        torch.cuda.synchronize()
        ex, ew = x.detach().clone().requires_grad_(), w0.clone().requires_grad_()
        ey = ops.layer_norm(ex, ew)
        assert all(torch.equal(p, q) for p, q in zip(out, (ey, *torch.autograd.grad(ey, (ex, ew), dy)))), i
        with torch.no_grad():
            x.mul_(0.5)


def test_calls_from_two_threads(cuda):
    """Two threads on two streams, forward and backward: each gets its own results."""
    import threading
    data = [[make(cuda, (600 + 40 * i, 96 + 32 * i), torch.bfloat16, 4 * i + j) for j in range(3)] for i in range(2)]

    def work(x, r, dy, seed):
        x, r = x.clone().requires_grad_(), r.clone().requires_grad_()
        y, z = ops.dropout_add_layer_norm(x, r, p=0.3, rng=(seed, 1))
        return (y.detach(), z.detach(), *torch.autograd.grad((y, z), (x, r), (dy, dy)))
    want = [work(*d, i) for i, d in enumerate(data)]
    torch.cuda.synchronize()
    got, bad = [None, None], []

    def run(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(30):
                    got[i] = work(*data[i], i)
                    torch.cuda.current_stream().synchronize()
                    assert all(torch.equal(a, b) for a, b in zip(got[i], want[i]))
        except BaseException as e:                                                   # noqa: BLE001
            bad.append(e)
    threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad, bad


def test_saved_tensors_go_through_hooks(cuda):
    """What the backward pass reads passes the saved-tensor hooks (offloading): gradients are the same."""
    x, w, dy = make(cuda, (33, 64), torch.bfloat16, 1).requires_grad_(), make(cuda, (64,), torch.float32, 2).requires_grad_(), make(cuda, (33, 64), torch.bfloat16, 3)
    want = torch.autograd.grad(ops.layer_norm(x, w), (x, w), dy)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.cpu(), lambda t: t.to(cuda)):
        y = ops.layer_norm(x, w)
    got = torch.autograd.grad(y, (x, w), dy)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_shared_heads_sum_their_gradients(cuda):
    """One key head expanded over the query heads: autograd sums what the expanded view gets."""
    B, T, H, D = 2, 9, 4, 32
    inv = ops.rotary_frequencies(D)[0].to(cuda)
    k, dk = make(cuda, (B, T, 1, D), torch.float32, 1).requires_grad_(), make(cuda, (B, T, H, D), torch.float32, 2)
    got, = torch.autograd.grad(ops.rotary(k.expand(B, T, H, D), 5, inv), k, dk)
    each = ops.rotary(k.detach(), 5, inv)
    assert torch.equal(ops.rotary(k.expand(B, T, H, D), 5, inv), each.expand(B, T, H, D))
    want = O.rotary(dk.cpu(), torch.arange(T) + 5, inv.cpu(), False, "bthd", 1.0, True).sum(2, keepdim=True)
    near(got, want, dk.cpu().double().abs().sum((2, 3), keepdim=True))


def test_captured_serving_step(cuda):
    """A token's norm and rotary positions in a graph whose positions move on between replays."""
    B, H, D = 6, 4, 64
    x, r = make(cuda, (B, H * D), torch.float16, 1), make(cuda, (B, H * D), torch.float16, 2)
    w = make(cuda, (H * D,), torch.float16, 3)
    inv = ops.rotary_frequencies(D)[0].to(cuda)
    pos = torch.arange(B, device=cuda).view(B, 1) * 1000

    def step():
        y, z = ops.dropout_add_layer_norm(x, r, w)
        return ops.rotary(y.view(B, 1, H, D), pos, inv), z
    with torch.no_grad():
        step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        for _ in range(4):
            graph.replay()
            torch.cuda.synchronize()
            eager = step()
            assert torch.equal(out[0], eager[0]) and torch.equal(out[1], eager[1])
            pos += 1


# ------------------------------------------------------------------------------------------------------------------ as they are used together
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_a_block_over_keypoint_tokens(cuda, dtype):
    """A transformer block over the keypoints of two frames: norm, joint projection, rotary positions from (x, y), attention (torch), residual with
    dropout and the next norm in one pass, a hidden layer with dropout, the last residual.  Results and every gradient against the same
    block in 64 bits."""
    dt = TYPES[dtype]
    B, T, H, Dh, p = 2, 37, 4, 32, 0.1
    D = H * Dh
    g = torch.Generator().manual_seed(4)
    P = {"w1": 1 + 0.1 * torch.randn(D, generator=g), "b1": 0.1 * torch.randn(D, generator=g), "w2": 1 + 0.1 * torch.randn(D, generator=g), "b2": 0.1 * torch.randn(D, generator=g),
         "qkv": torch.randn(D, 3 * D, generator=g) / D ** 0.5, "out": torch.randn(D, D, generator=g) / D ** 0.5, "up": torch.randn(D, 2 * D, generator=g) / D ** 0.5,
         "down": torch.randn(2 * D, D, generator=g) / (2 * D) ** 0.5}
    P = {k: (v if k in ("w1", "b1", "w2", "b2") else v.to(dt).float()) for k, v in P.items()}
    x0 = torch.randn(B, T, D, generator=g).to(dt)
    xy = torch.rand(B, T, 2, generator=g) * 639
    inv, _ = ops.rotary_frequencies(Dh, 100.0, axes=2)
    dy = torch.randn(B, T, D, generator=g).to(dt)
    seeds = [(5, 0), (5, 1), (5, 2)]

    def attend(q, k, v):
        s = torch.matmul(q, k.transpose(-1, -2).contiguous()) / Dh ** 0.5
        return torch.matmul(torch.softmax(s, -1), v)

    def block(x, P, norm, fused, drop, turn):
        h = norm(x, P["w1"], P["b1"])
        q, k, v = torch.matmul(h, P["qkv"].to(h.dtype)).view(B, T, 3, H, Dh).unbind(2)
        q, k = turn(q, k)
        a = attend(*(t.transpose(1, 2).contiguous().to(torch.float64 if x.dtype == torch.float64 else torch.float32) for t in (q, k, v)))
        a = torch.matmul(a.transpose(1, 2).reshape(B, T, D).to(h.dtype), P["out"].to(h.dtype))
        y, z = fused(a, x, P["w2"], P["b2"], seeds[0])
        u = drop(torch.relu(torch.matmul(y, P["up"].to(y.dtype))), seeds[1], None)
        return drop(torch.matmul(u, P["down"].to(y.dtype)), seeds[2], z)

    leaf = x0.to(cuda).requires_grad_()
    Pd = {k: v.to(cuda).requires_grad_() for k, v in P.items()}
    got = block(leaf, Pd, ops.layer_norm, lambda a, x, w, b, s: ops.dropout_add_layer_norm(a, x, w, b, p=p, rng=s), lambda t, s, r: ops.dropout(t, p, s, residual=r),
                lambda q, k: ops.rotary(q, xy.to(cuda), inv.to(cuda), k=k))
    got_g = torch.autograd.grad(got, (leaf, *Pd.values()), dy.to(cuda))

    def drop64(t, s, r):
        keep = O.keep_mask(t.numel(), p, *s).view(t.shape).double() * O.drop_scale(p)
        return t * keep + (0.0 if r is None else r)

    def norm64(x, w, b):
        d = x - x.mean(-1, keepdim=True)
        return d / (d.square().mean(-1, keepdim=True) + 1e-5).sqrt() * w + b

    def turn64(*ts):
        angle = torch.cat([xy[..., :1].double() * inv[:Dh // 4], xy[..., 1:].double() * inv[Dh // 4:]], -1).unsqueeze(2)
        c, s = angle.cos(), angle.sin()
        return [torch.cat([t[..., :Dh // 2] * c - t[..., Dh // 2:] * s, t[..., Dh // 2:] * c + t[..., :Dh // 2] * s], -1) for t in ts]

    def fused64(a, x, w, b, s):
        z = drop64(a, s, x)
        return norm64(z, w, b), z
    ref = x0.double().requires_grad_()
    P64 = {k: v.double().requires_grad_() for k, v in P.items()}
    want = block(ref, P64, norm64, fused64, drop64, turn64)
    want_g = torch.autograd.grad(want, (ref, *P64.values()), dy.double())
    # relative 2-norm: some 30 roundings of the type in a chain, each half a step, at random: sqrt(30) * eps / 2, three times that as the bar
    # (fp32: the library's products sum 256 terms, another factor of 16)
    bar = 3 * math.sqrt(30) * torch.finfo(dt).eps / 2 * (16 if dtype == "f32" else 1)
    for name, a, b in zip(("y", "x", *P), (got, *got_g), (want, *want_g)):
        rel = float((a.detach().cpu().double() - b.detach()).norm() / b.detach().norm())
        assert rel <= bar, (name, rel, bar)


# ------------------------------------------------------------------------------------------------------------------ calls that other machinery watches
def test_traced_calls_are_refused_on_the_device(cuda):
    """Forward and backward under a tracer; under a mode that only watches, the call runs as ever."""
    from torch.fx.experimental.proxy_tensor import make_fx
    from torch.utils.flop_counter import FlopCounterMode
    x, dy = make(cuda, (9, 64), torch.bfloat16, 1), make(cuda, (9, 64), torch.bfloat16, 2)
    inv = ops.rotary_frequencies(64)[0].to(cuda)
    for f in (lambda t: ops.layer_norm(t), lambda t: ops.dropout_add_layer_norm(t, t, p=0.5, rng=(1, 2))[0], lambda t: ops.dropout(t, 0.5, (1, 2)),
              lambda t: ops.rotary(t.view(1, 9, 1, 64), 3, inv).view(9, 64)):
        with pytest.raises(_hip.YpError, match="cannot be traced"):
            torch.jit.trace(f, x)
        with pytest.raises(_hip.YpError, match="cannot be traced"):
            make_fx(f)(x)
        leaf = x.clone().requires_grad_()
        y = f(leaf)
        with pytest.raises(RuntimeError, match="cannot be traced"):
            make_fx(lambda g: torch.autograd.grad(y, leaf, g, retain_graph=True)[0])(dy)
        want = torch.autograd.grad(y, leaf, dy)[0]
        with FlopCounterMode(display=False):
            again = f(leaf)
            got, = torch.autograd.grad(again, leaf, dy)
        assert torch.equal(again, y) and torch.equal(got, want)


def test_operands_without_memory_are_refused(cuda):
    """A wrapper beside ordinary tensors must not pass for an operand that was not given; a tensor that torch knows to be zero is one of zeros."""
    from test_token_ops import Wrapper

    def hollow(t):
        return Wrapper(t.shape, t.dtype, t.device)
    x, r, w = make(cuda, (4, 8), torch.float32, 1), make(cuda, (4, 8), torch.float32, 2), make(cuda, (8,), torch.float32, 3)
    q, at, inv, state = make(cuda, (1, 4, 2, 8), torch.float32, 4), torch.arange(4, device=cuda), ops.rotary_frequencies(8)[0].to(cuda), torch.tensor([1, 2], device=cuda)
    for call in (lambda: ops.layer_norm(x, hollow(w)), lambda: ops.layer_norm(x, None, hollow(w)), lambda: ops.dropout(x, 0.5, hollow(state)), lambda: ops.dropout(x, 0.5, (1, 2), residual=hollow(x)),
                 lambda: ops.dropout_add_layer_norm(x, hollow(x)), lambda: ops.dropout_add_layer_norm(x, r, hollow(w)), lambda: ops.dropout_add_layer_norm(x, r, p=0.5, rng=hollow(state)),
                 lambda: ops.rotary(q, hollow(at), inv), lambda: ops.rotary(q, at, hollow(inv)), lambda: ops.rotary(q, at, inv, k=hollow(q)), lambda: ops.rotary(hollow(q), at, inv)):
        with pytest.raises(_hip.YpError):
            call()
    zero = torch._efficientzerotensor((4, 8), device=cuda)
    assert zero.data_ptr() == 0
    none = torch.zeros(4, 8, device=cuda)
    assert torch.equal(ops.dropout_add_layer_norm(x, zero)[1], x) and torch.equal(ops.dropout(zero, 0.5, (1, 2), residual=r), r) and torch.equal(ops.layer_norm(zero), none)
    assert not ops.rotary(zero.view(1, 4, 1, 8), at, inv).any()
    a, b = x.clone().requires_grad_(), r.clone().requires_grad_()
    y, z = ops.dropout_add_layer_norm(a, b, p=0.5, rng=(1, 2))
    want = torch.autograd.grad((y, z), (a, b), (none, x), retain_graph=True)
    assert all(torch.equal(i, j) for i, j in zip(torch.autograd.grad((y, z), (a, b), (zero, x), retain_graph=True), want))
    want = torch.autograd.grad((y, z), (a, b), (x, none), retain_graph=True)
    assert all(torch.equal(i, j) for i, j in zip(torch.autograd.grad((y, z), (a, b), (x, zero)), want))


def test_a_state_that_is_not_read_may_move_on(cuda):
    """Rates of 0 (or below half a step) draw nothing: the state may be written between forward and backward."""
    x, r, dy = (make(cuda, (7, 24), torch.bfloat16, i) for i in range(3))
    for p in (0.0, 1e-6):
        for f in (lambda a, s: ops.dropout(a, p, s), lambda a, s: ops.dropout(a, p, s, residual=r), lambda a, s: ops.dropout_add_layer_norm(a, r, p=p, rng=s)[1]):
            state, leaf = torch.tensor([3, 4], device=cuda), x.clone().requires_grad_()
            y = f(leaf, state)
            state[1] += 1
            assert torch.equal(torch.autograd.grad(y, leaf, dy)[0], dy)


def test_rotary_in_place_beside_each_other(cuda):
    """q and k of one tensor, side by side at any depth, share no element: turned in place; what meets stays refused."""
    B, T, H, D = 2, 5, 4, 16
    inv, at = ops.rotary_frequencies(D)[0].to(cuda), torch.arange(T, device=cuda) + 7

    def turned(joint, q, k, layout="bthd"):
        """q, k: functions of the joint tensor"""
        want = ops.rotary(q(joint), at, inv, k=k(joint), layout=layout)
        rest = joint.clone()
        q(rest).zero_(), k(rest).zero_()
        ops.rotary(q(joint), at, inv, k=k(joint), layout=layout, inplace=True)
        assert torch.equal(q(joint), want[0]) and torch.equal(k(joint), want[1])
        q(joint).zero_(), k(joint).zero_()
        assert torch.equal(joint, rest)                                              # nothing but q and k was written
    for i, j in ((0, 1), (1, 0), (2, 0), (1, 2)):
        turned(make(cuda, (B, T, H, 3, D), torch.bfloat16, 1), lambda t: t[..., i, :], lambda t: t[..., j, :])            # beside each other in a head
        turned(make(cuda, (B, T, 3, H, D), torch.float32, 2), lambda t: t[:, :, i], lambda t: t[:, :, j])                # in a token
        turned(make(cuda, (T, B, 3, H, D), torch.bfloat16, 3), lambda t: t[:, :, i].transpose(0, 1), lambda t: t[:, :, j].transpose(0, 1))
        turned(make(cuda, (B, 3, H, T, D), torch.float16, 4), lambda t: t[:, i], lambda t: t[:, j], "bhtd")              # in a batch entry
        turned(make(cuda, (B, H, T, 3, D), torch.float16, 5), lambda t: t[..., i, :], lambda t: t[..., j, :], "bhtd")
    turned(make(cuda, (B, T, 2, 3, D), torch.bfloat16, 6), lambda t: t[:, :, 0:1, :2].flatten(2, 3), lambda t: t[:, :, 1, 2:], "bthd")     # head numbers 2 and 1
    turned(make(cuda, (B, T, H, 3 * D), torch.bfloat16, 7), lambda t: t[:, :, :, 3:3 + D], lambda t: t[:, :, :2, 2 * D:])                  # every head of q, the first two of k
    odd = make(cuda, (B, T, H, 3 * D), torch.bfloat16, 8)
    clean = odd.clone()
    for q, k in ((odd[..., :D], odd[..., D // 2:D // 2 + D]), (odd[..., :D], odd[..., :D]), (odd[:, :, :2, :D], odd[:, :, 1:3, :D]), (odd[..., D:2 * D], odd[:, :, 1:, D:2 * D]),
                 (odd[..., 2 * D:], odd.flatten()[3 * D - 8:][:B * T * H * 2 * D].view(B, T, H, 2 * D)[..., :D])):
        with pytest.raises(_hip.YpError):
            ops.rotary(q, at, inv, k=k, inplace=True)
    assert torch.equal(odd, clean)
    q, k = odd[:, :, :0, :D], odd[..., :D]                                           # no head of q: nothing to meet
    want = ops.rotary(k, at, inv)
    ops.rotary(q, at, inv, k=k, inplace=True)
    assert torch.equal(k, want)


# ------------------------------------------------------------------------------------------------------------------ rows far from zero
def far_rows(D, dt, seed=1):
    """Rows whose values say little beside their mean: constant ones, ones that leave their constant in one place, steps of the type around 1024."""
    step = torch.finfo(dt).eps
    g = torch.Generator().manual_seed(seed + D)
    x = torch.empty(10, D, dtype=torch.float64)
    for i, v in enumerate((13696.0, -13696.0, 1368.0, 7.25, 40000.0, 0.0)):
        x[i] = v
    x[6] = 13696.0
    x[6, D // 2] += 8192 * step
    x[7] = 1368.0
    x[7, -1] -= 1024 * step
    x[8:] = 1024.0 * (1.0 + step * torch.randint(0, 3, (2, D), generator=g).double())
    return x.to(dt)


def centred_error(x, eps):
    """What x - mean and 1 / deviation may be off by, (in deviations, relative): the mean is a sum of at most 30 roundings, and their result is summed and
    taken off with at most 30 again, so that a rounding of the mean's size enters in its square only."""
    n = 32 * 2.0 ** -24
    _, mean, rstd, xhat = O.layer_norm(x, None, None, eps)
    first = n * x.double().abs().mean(-1, keepdim=True)
    return n * ((x.double() - mean).abs().mean(-1, keepdim=True) + first) * rstd, n * (1.0 + 2.0 * (first * rstd).square()) + 8 * 2.0 ** -24


FAR_WIDTHS = [1, 7, 28, 60, 100, 777, 1000, 1091, 4100, 9000, 12345]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", FAR_WIDTHS)
def test_layer_norm_of_rows_that_hardly_vary(cuda, D, dtype):
    """The rounding of the mean must not become the result where eps alone makes the deviation."""
    dt = TYPES[dtype]
    x, w, b = far_rows(D, dt), make(cuda, (D,), torch.float32, 3), make(cuda, (D,), torch.float32, 4)
    shift, scale = centred_error(x, 1e-5)
    _, _, _, xhat = O.layer_norm(x, None, None, 1e-5)
    off = shift + xhat.abs() * scale
    near(ops.layer_norm(x.to(cuda)), xhat, 0.0, off)
    wc, bc = w.cpu().double(), b.cpu().double()
    near(ops.layer_norm(x.to(cuda), w, b), xhat * wc + bc, 0.0, off * wc.abs() + 2 * 2.0 ** -24 * ((xhat * wc).abs() + bc.abs()))
    y, z = ops.dropout_add_layer_norm(torch.zeros_like(x).to(cuda), x.to(cuda))
    assert torch.equal(z.cpu(), x)
    near(y, xhat, 0.0, off)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [2, 60, 777, 5000, 16384])
def test_layer_norm_of_a_constant_that_one_value_leaves(cuda, D, dtype):
    """The lone value is far below the others, so that no fp32 sum holds all digits: bf16, which takes the exact sum's remainder for the rounding of the
    mean, may be off by the sum's own rounding (30 steps of the mean, whose size is sqrt(D) deviations at the most)."""
    dt = TYPES[dtype]
    x = torch.full((3, D), 13696.0, dtype=torch.float64)
    x[0, 0], x[1, D // 2], x[2, -1] = 2.0 ** -9 * 1.5, -(2.0 ** -7), 0.0
    x = x.to(dt)
    shift, scale = centred_error(x, 1e-5)
    _, _, rstd, xhat = O.layer_norm(x, None, None, 1e-5)
    sums = 32 * 2.0 ** -24 * x.double().abs().mean(-1, keepdim=True) * rstd if dtype == "bf16" else 0.0
    near(ops.layer_norm(x.to(cuda)), xhat, 0.0, shift + xhat.abs() * scale + sums)


def centred_backward(x, w, dy, eps):
    """-> (dx, error), (dweight, error) on rows far from zero: xhat's own error as in centred_error, sums of 32 roundings, some eight operations a value."""
    u = 2.0 ** -24
    shift, scale = centred_error(x, eps)
    _, _, rstd, xhat = O.layer_norm(x, None, None, eps)
    dx, dw, _ = O.layer_norm_backward(x, w, dy, eps)
    ex = shift + xhat.abs() * scale
    h = (dy.double() * w.double()).abs()
    m1, m2, moved = h.mean(-1, keepdim=True), (h * xhat.abs()).mean(-1, keepdim=True), (h * ex).mean(-1, keepdim=True)
    terms = h + m1 + xhat.abs() * m2
    dx_error = rstd * (xhat.abs() * (32 * u * m2 + moved) + ex * (m2 + moved) + 32 * u * m1 + (8 * u + scale) * terms)
    dw_error = (dy.double().abs() * (ex + 2 * F32 * xhat.abs())).sum(0)
    return (dx, dx_error), (dw, dw_error)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", FAR_WIDTHS)
def test_layer_norm_backward_of_rows_that_hardly_vary(cuda, D, dtype):
    """The backward pass has the forward pass's xhat, not one that the rounding of mean / deviation went into: constant rows give dweight nothing."""
    dt = TYPES[dtype]
    x, dy, w = far_rows(D, dt), make("cpu", (10, D), dt, 5, 0.1, 0.7), make("cpu", (D,), torch.float32, 3, 1.0, 0.3)
    (dx, dx_error), (dw, dw_error) = centred_backward(x, w, dy, 1e-5)
    leaf, weight = x.to(cuda).requires_grad_(), w.to(cuda).requires_grad_()
    got = torch.autograd.grad(ops.layer_norm(leaf, weight), (leaf, weight), dy.to(cuda))
    near(got[0], dx, 0.0, dx_error)
    near(got[1], dw, 0.0, dw_error)
    for p in (0.0, 0.25):
        branch = torch.zeros_like(x).to(cuda).requires_grad_()
        y, z = ops.dropout_add_layer_norm(branch, leaf, weight, p=p, rng=(1, 2))
        dbranch, dres, dweight = torch.autograd.grad((y, z), (branch, leaf, weight), (dy.to(cuda), torch.zeros_like(z)))
        keep = O.keep_mask(10 * D, p, 1, 2).view(10, D).double() * O.drop_scale(p)
        near(dbranch, dx * keep, 0.0, (dx_error + 2 * 2.0 ** -24 * dx.abs()) * keep)
        near(dres, dx, 0.0, dx_error)
        near(dweight, dw, 0.0, dw_error)


@pytest.mark.parametrize("D", [64, 777, 2000, 9001])
def test_layer_norm_backward_far_from_zero(cuda, D):
    """f32 rows of mean 1000 and deviation 0.01, and of mean 4096 and deviation 1: forward and backward."""
    x = torch.cat([make("cpu", (200, D), torch.float32, 1, 1000.0, 0.01), make("cpu", (200, D), torch.float32, 2, -4096.0, 1.0)])
    dy, w = make("cpu", (400, D), torch.float32, 5, 0.1, 0.7), make("cpu", (D,), torch.float32, 3, 1.0, 0.3)
    (dx, dx_error), (dw, dw_error) = centred_backward(x, w, dy, 1e-5)
    leaf, weight = x.to(cuda).requires_grad_(), w.to(cuda).requires_grad_()
    got = torch.autograd.grad(ops.layer_norm(leaf, weight), (leaf, weight), dy.to(cuda))
    near(got[0], dx, 0.0, dx_error)
    near(got[1], dw, 0.0, dw_error)


def test_layer_norm_statistics_at_the_entry_points(cuda):
    """Both forms of the statistics: with `stats`, xhat is as exact as in y; with mean and rstd it carries half a step of the mean, and no more."""
    l, (rows, D) = _hip.lib(), (6, 300)
    x, dy = make(cuda, (rows, D), torch.float32, 1, 1000.0, 0.01), make(cuda, (rows, D), torch.float32, 2)
    x[5] = 13730.0
    y, dx, dw, stats = torch.empty_like(x), torch.empty_like(x), torch.empty(D, device=cuda), torch.empty(rows, 3, device=cuda)
    nb = l.yp_layer_norm_bwd_workspace_bytes(rows, D, _hip.YP_F32)
    ws = torch.empty(nb, dtype=torch.uint8, device=cuda)
    _, mean, rstd, _ = O.layer_norm(x.cpu(), None, None, 1e-5)
    one = torch.ones(D)
    (want, error), (want_w, error_w) = centred_backward(x.cpu(), one, dy.cpu(), 1e-5)
    step = 2.0 ** -24 * mean.abs() * rstd                                            # (the nearest number is half a step away: 2^-24 of it)
    m1 = dy.cpu().double().abs().mean(-1, keepdim=True)
    m2 = (dy.cpu().double() * O.layer_norm(x.cpu(), None, None, 1e-5)[3]).abs().mean(-1, keepdim=True)
    xhat = O.layer_norm(x.cpu(), None, None, 1e-5)[3].abs()
    for rest in (True, False):
        how = dict(rows=rows, D=D, dtype=_hip.YP_F32, wdtype=_hip.YP_F32, eps=1e-5, x=x.data_ptr(), x_stride=D,
                   **(dict(stats=stats.data_ptr()) if rest else dict(mean=stats.view(-1)[:rows].data_ptr(), rstd=stats.view(-1)[rows:].data_ptr())))
        stats.fill_(7.0)
        _hip.check(l.yp_layer_norm_fwd(C.byref(_hip.YpLayerNormDesc(y=y.data_ptr(), **how)), _hip.stream_ptr()))
        nearest = (stats[:, 0] if rest else stats.view(-1)[:rows]).cpu().double()
        assert bool(((nearest - mean.view(-1)).abs() <= 2.0 ** -24 * mean.view(-1).abs() * 1.001).all())
        if rest:
            assert bool(((nearest + stats[:, 2].cpu().double() - mean.view(-1)).abs() <= 2.0 ** -36 * mean.view(-1).abs()).all())
        else:
            assert bool((stats.view(-1)[2 * rows:] == 7.0).all())
        _hip.check(l.yp_layer_norm_bwd(C.byref(_hip.YpLayerNormDesc(dy=dy.data_ptr(), dy_stride=D, dres=dx.data_ptr(), dweight=dw.data_ptr(), workspace=ws.data_ptr(),
                                                                    workspace_bytes=nb, **how)), _hip.stream_ptr()))
        s = 0.0 if rest else step
        near(dx, want, 0.0, error + rstd * s * (m2 + xhat * m1 + 2 * s * m1))
        near(dw, want_w, 0.0, error_w + (dy.cpu().double().abs() * s).sum(0))


# ------------------------------------------------------------------------------------------------------------------ what no one asked for
def test_frozen_inputs_cost_the_backward_pass_no_tensors(cuda):
    """Gradients of the rows are written where they are wanted only: each set of leaves gets the full pass's rows bit for bit, the weights' sums (over other
    workgroups' parts, as the kernels differ) within their bound, and no more memory than its gradients."""
    rows, D = 8192, 1000
    x, r, dy, dz = (make(cuda, (rows, D), torch.bfloat16, i) for i in range(4))
    w, b = make(cuda, (D,), torch.float32, 5), make(cuda, (D,), torch.float32, 6)
    size = rows * D * 2
    # beside the gradients: the partial sums, the weights' gradients, and what torch's allocator hands out unsplit (up to 1 MiB a buffer, five at the most)
    sums = _hip.lib().yp_layer_norm_bwd_workspace_bytes(rows, D, _hip.YP_BF16) + 64 * D + (5 << 20)
    assert sums < size                                                               # (a tensor too many shows)
    for p in (0.0, 0.3):
        full = None
        for want in range(15, 0, -1):
            leaves = [t.clone().requires_grad_(bool(want >> i & 1)) for i, t in enumerate((x, r, w, b))]
            asked = [t for t in leaves if t.requires_grad]
            for with_z in (True, False):
                y, z = ops.dropout_add_layer_norm(*leaves, p=p, rng=(1, 2))
                outs, grads = ((y, z), (dy, dz)) if with_z else ((y,), (dy,))
                torch.cuda.synchronize()
                before = torch.cuda.memory_allocated()
                torch.cuda.reset_peak_memory_stats()
                got = torch.autograd.grad(outs, asked, grads)
                torch.cuda.synchronize()
                peak = torch.cuda.max_memory_allocated() - before
                # (x and the residual share one gradient where nothing is dropped; where something is, the residual's is written with x's)
                tensors = (0, 2, 1, 2)[want & 3] if p else int(want & 3 != 0)
                assert peak <= tensors * size + sums, (p, want, with_z, peak, tensors * size, sums)
                if want == 15:
                    full = full or {}
                    full[with_z] = got
                    _, dw, db = norm_backward_bound(z.detach().cpu(), w.cpu(), dy.cpu(), 1e-5)
                for a, i in zip(got, [i for i in range(4) if want >> i & 1]):
                    if i < 2:
                        assert torch.equal(a, full[with_z][i])
                    else:
                        near(a, *(dw, db)[i - 2])
    leaf = x.clone().requires_grad_()                                                # y unused: z's gradient goes through, in no pass over z
    y, z = ops.dropout_add_layer_norm(r, leaf, w, b, p=0.3, rng=(1, 2))
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    assert torch.equal(torch.autograd.grad(z, leaf, dz)[0], dz)
    assert torch.cuda.max_memory_allocated() - before < size


FIRST_CALL = """
import torch
from yolopoint_amd.utils import token_ops as ops
cuda, D = torch.device("cuda:0"), 16000
g = torch.Generator().manual_seed(1)
x0, dy, w0 = (torch.randn(s, generator=g).half().to(cuda) for s in ((7, D), (7, D), (D,)))
st = torch.cuda.Stream()
st.wait_stream(torch.cuda.current_stream())
with torch.cuda.stream(st):
    x, w = x0.clone().requires_grad_(), w0.clone().requires_grad_()
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph, stream=st):
    y = ops.layer_norm(x, w)
    out = (y.detach(), *torch.autograd.grad(y, (x, w), dy))
for i in range(3):
    graph.replay()
    torch.cuda.synchronize()
    ex, ew = x.detach().clone().requires_grad_(), w0.clone().requires_grad_()
    ey = ops.layer_norm(ex, ew)
    assert all(torch.equal(p, q) for p, q in zip(out, (ey, *torch.autograd.grad(ey, (ex, ew), dy)))), i
    with torch.no_grad():
        x.mul_(0.5)
torch.cuda.synchronize()
print("captured first call: ok")
"""


def test_captured_first_call_in_a_process_of_its_own(cuda):
    """The captured call is the process's first of these kernels, so that what the launch asks the runtime for (a larger LDS limit, the occupancy) is asked
    inside the capture."""
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", FIRST_CALL], capture_output=True, text=True, timeout=100, cwd=root)
    assert r.returncode == 0 and "captured first call: ok" in r.stdout, r.stderr[-2000:]
