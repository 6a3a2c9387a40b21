"""Layer norm, rotary positions and gradient clipping on the GPU against plain formulas in 64 bits.

Tolerances count roundings: half a step of the result's type, and u = 2^-24 per fp32 operation on the terms that enter a result."""
import math

import pytest
import torch

from q38 import ops

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def half_step(t):
    return torch.finfo(t).eps / 2


def within(got, want, tol, what):
    """Every element within its tolerance; a type's smallest step covers results near zero."""
    off = (got.double() - want).abs() - tol - torch.finfo(got.dtype).tiny * 2
    assert not (off > 0).any() and not got.isnan().any(), (what, off.max().item(), int((off > 0).sum()))


# ---- layer norm ---------------------------------------------------------------------------------------------------------------
def norm_formula(x, w, b, dy, eps):
    """y, dx, dw, db in 64 bits, and the sums of magnitudes that fp32 roundings are counted on."""
    x, dy = x.double().reshape(-1, x.shape[-1]), dy.double().reshape(-1, x.shape[-1])
    w = torch.ones_like(x[0]) if w is None else w.double()
    b = torch.zeros_like(x[0]) if b is None else b.double()
    mu = x.mean(-1, keepdim=True)
    r = 1 / torch.sqrt((x - mu).square().mean(-1, keepdim=True) + eps)
    hat = (x - mu) * r
    g = dy * w
    mean = lambda t: t.mean(-1, keepdim=True)
    hat_size = hat.abs() + mean(x.abs()) * r                      # a rounding of mu or of x - mu is one of |x|
    y_size = hat_size * w.abs() + b.abs()
    dx = r * (g - mean(g) - hat * mean(g * hat))
    dx_size = r * (g.abs() + mean(g.abs()) + hat_size * mean(g.abs() * hat_size))
    return (hat * w + b, dx, (dy * hat).sum(0), dy.sum(0)), (y_size, dx_size, (dy.abs() * hat_size).sum(0), dy.abs().sum(0))


def check_norm(x, w, b, dy, eps=1e-5, out_dtype=None):
    rows = x.numel() // x.shape[-1]
    leaves = [t.detach().requires_grad_() for t in (x, w, b) if t is not None]
    args = iter(leaves)
    y = ops.layer_norm(next(args), None if w is None else next(args), None if b is None else next(args), eps, out_dtype)
    assert y.shape == x.shape and y.dtype == (out_dtype or x.dtype)
    grads = torch.autograd.grad(y, leaves, dy)
    want, size = norm_formula(x, w, b, dy, eps)
    # a mean: up to 32 additions in a thread, ten in trees, one division, twice; the square root and the products around it eight more
    sums = 80 * U
    within(y.reshape(want[0].shape), want[0], half_step(y.dtype) * want[0].abs() + sums * size[0], "y")
    within(grads[0].reshape(want[1].shape), want[1], half_step(x.dtype) * want[1].abs() + 2 * sums * size[1], "dx")
    got = iter(grads[1:])
    order = rows / 148 + 64                                        # additions in the longest chain: rows of a group, groups, CTAs
    for p, e, s, name in ((w, want[2], size[2], "dw"), (b, want[3], size[3], "db")):
        if p is not None:
            g = next(got)
            assert g.dtype == p.dtype
            within(g, e, half_step(p.dtype) * e.abs() + (order + 80) * U * s, name)
    with torch.no_grad():
        assert torch.equal(ops.layer_norm(x, w, b, eps, out_dtype), y)


# widths: one element, a part of a warp, each kind of row (a warp with 8, 16 and 32 elements per thread; groups; 16 per thread; sums in shared memory; longer
# than registers hold) at its ends, odd ones between; rows: none of a group's, one more than a CTA's, several rounds of the grid
NORM_SHAPES = [(1, 1), (3, 7), (1, 64), (33, 256), (9, 257), (2500, 96), (17, 512), (5, 513), (6000, 520), (130, 1024), (64, 1025), (5, 2305), (700, 2048), (9, 4096), (7, 4097),
               (3, 8192), (5, 8193), (2, 16384), (301, 8200), (2, 16385), (3, 20001), (100_003, 8), (70_000, 5)]


@pytest.mark.parametrize("rows,dim", NORM_SHAPES)
@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_layer_norm_shapes(rows, dim, dtype):
    gen = torch.Generator(device="cuda").manual_seed(rows * 31 + dim)
    rand = lambda *s: torch.randn(*s, device="cuda", generator=gen)
    check_norm((rand(rows, dim) * 2 + 1).to(dtype), 1 + 0.5 * rand(dim), rand(dim), rand(rows, dim).to(dtype))


@pytest.mark.parametrize("dtype,param,out,affine", [(FP16, FP32, None, "wb"), (FP16, FP16, None, "wb"), (BF16, BF16, None, "wb"), (FP32, FP32, BF16, "wb"), (FP32, BF16, BF16, "w"),
                                                    (BF16, FP32, None, "b"), (FP32, FP16, None, "b"), (BF16, FP32, None, ""), (FP32, FP32, FP32, "")])
@pytest.mark.parametrize("dim", [72, 1031])
def test_layer_norm_types(dtype, param, out, affine, dim):
    gen = torch.Generator(device="cuda").manual_seed(dim)
    rand = lambda *s: torch.randn(*s, device="cuda", generator=gen)
    check_norm(rand(41, dim).to(dtype), rand(dim).to(param) if "w" in affine else None, rand(dim).to(param) if "b" in affine else None, rand(41, dim).to(out or dtype), out_dtype=out)


def test_layer_norm_far_from_zero():
    """The centred variance: a mean a thousand times the spread."""
    gen = torch.Generator(device="cuda").manual_seed(5)
    rand = lambda *s: torch.randn(*s, device="cuda", generator=gen)
    check_norm(1000 + rand(50, 640), rand(640), rand(640), rand(50, 640))
    flat = torch.full((3, 640), 2.5, device="cuda")                  # no spread at all: the result is the bias
    assert torch.equal(ops.layer_norm(flat, None, torch.ones(640, device="cuda")), torch.ones(3, 640, device="cuda"))


def test_layer_norm_strides_and_offsets():
    gen = torch.Generator(device="cuda").manual_seed(6)
    rand = lambda *s: torch.randn(*s, device="cuda", generator=gen)
    wide = rand(2, 9, 3, 200).to(BF16)
    w, b = rand(131)[1:129], rand(256)[::2]                          # not on 16 bytes; not contiguous
    for x in (wide[..., :128], wide[..., 1:129], wide[:, :, 1, 8:136], wide[..., :128].transpose(0, 2), rand(128, 40).to(BF16).t()):
        check_norm(x, w, b, rand(*x.shape).to(BF16))
    x = rand(6, 128)
    base = x.clone().requires_grad_()
    dy = rand(128).expand(6, 128)                                    # the gradient of a sum over rows: rows share memory
    y = ops.layer_norm(base, w, b)
    dx, = torch.autograd.grad(y, base, dy)
    want, size = norm_formula(x, w, b, dy, 1e-5)
    within(dx, want[1], 200 * U * size[1] + half_step(FP32) * want[1].abs(), "dx")
    xt = rand(5, 128)
    row = xt[:1].clone().requires_grad_()                            # a broadcast input: its gradient is the sum over copies
    g, = torch.autograd.grad(ops.layer_norm(row.expand(5, 128), w, b), row, xt)
    want, size = norm_formula(row.detach().expand(5, 128), w, b, xt, 1e-5)
    within(g, want[1].sum(0, keepdim=True), 250 * U * size[1].sum(0, keepdim=True), "row")


def test_layer_norm_of_tiny_values_without_eps():
    """A spread of 1e-18: its inverse is finite in fp32, the square of that is not."""
    gen = torch.Generator(device="cuda").manual_seed(7)
    rand = lambda *s: torch.randn(*s, device="cuda", generator=gen)
    for dim in (256, 777, 1500):
        x, dy = 1e-18 * rand(6, dim), rand(6, dim)
        leaf = x.requires_grad_()
        y = ops.layer_norm(leaf, eps=0.0)
        want, size = norm_formula(x.detach(), None, None, dy, 0.0)
        # Squares under the smallest normal number, 2^-126, count as zero: the variance v (about 1e-36) loses at most that, so 1 / sqrt(v) is off by at most
        # 0.51 * 2^-126 / v of itself (v (1 - a))^-1/2 = v^-1/2 (1 + a / 2 + ...), a < 0.02), and with it each of the up to three factors 1 / sqrt(v) in dx
        lost = 0.51 * 2.0 ** -126 / x.detach().double().var(-1, unbiased=False, keepdim=True)
        assert lost.max() < 0.01
        within(y, want[0], (100 * U + lost) * size[0], "y")
        within(torch.autograd.grad(y, leaf, dy)[0], want[1], (200 * U + 3.1 * lost) * size[1], "dx")


def test_layer_norm_empty_and_not_finite():
    w = torch.ones(64, device="cuda", requires_grad=True)
    x = torch.zeros(0, 64, device="cuda", dtype=BF16, requires_grad=True)
    y = ops.layer_norm(x, w, w)
    dx, dw = torch.autograd.grad(y, [x, w], torch.zeros(0, 64, device="cuda", dtype=BF16))
    assert y.shape == dx.shape == (0, 64) and not dw.any()
    for bad in (float("nan"), float("inf")):                         # stays in its row, and in the weight's gradient
        for dim in (64, 2000):
            x = torch.randn(40, dim, device="cuda")
            clean = ops.layer_norm(x)
            x[7, 3] = bad
            x.requires_grad_()
            w = torch.ones(dim, device="cuda", requires_grad=True)
            y = ops.layer_norm(x, w)
            keep = torch.arange(40, device="cuda") != 7
            assert torch.equal(y[keep], clean[keep]) and y[7].isnan().any()
            dx, dw = torch.autograd.grad(y, [x, w], torch.ones_like(y))
            assert dx[keep].isfinite().all() and dx[7].isnan().all() and dw.isnan().any()


def test_layer_norm_only_what_is_wanted_and_same_bits():
    gen = torch.Generator(device="cuda").manual_seed(8)
    rand = lambda *s: torch.randn(*s, device="cuda", generator=gen)
    x, w, b, dy = rand(3000, 384), rand(384), rand(384), rand(3000, 384)
    full = [t.clone().requires_grad_() for t in (x, w, b)]
    first = torch.autograd.grad(ops.layer_norm(*full), full, dy)
    again = torch.autograd.grad(ops.layer_norm(*full), full, dy)
    assert all(torch.equal(a, c) for a, c in zip(first, again))
    for i in range(3):
        some = [t.clone().requires_grad_(k == i) for k, t in enumerate((x, w, b))]
        one, = torch.autograd.grad(ops.layer_norm(*some), [some[i]], dy)
        assert torch.equal(one, first[i])
    only_b = b.clone().requires_grad_()
    g, = torch.autograd.grad(ops.layer_norm(x, None, only_b), only_b, dy)      # without a weight the bias is the second tensor
    assert torch.equal(g, first[2])
    y = ops.layer_norm(full[0], w, b)
    with pytest.raises(RuntimeError, match="gradient of the gradient"):
        torch.autograd.grad(y, full[0], dy, create_graph=True)
    x2 = x.clone().requires_grad_()
    h = x2 * 1.0
    y = ops.layer_norm(h, w, b)
    h.mul_(2)                                                        # a saved input that changed is noticed
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_layer_norm_gradient_by_differences():
    """Directional derivatives of the kernel's own forward; a step of 2^-6 leaves (2^-6)^2 of third derivatives, roundings add 2^-24 / 2^-6."""
    gen = torch.Generator(device="cuda").manual_seed(9)
    rand = lambda *s: torch.randn(*s, device="cuda", generator=gen)
    args = [rand(4, 96).requires_grad_(), rand(96).requires_grad_(), rand(96).requires_grad_()]
    dy = rand(4, 96)
    grads = torch.autograd.grad(ops.layer_norm(*args), args, dy)
    for i in range(3):
        v = rand(*args[i].shape)
        h = 2.0 ** -6
        moved = [[a.detach() + s * h * v if k == i else a.detach() for k, a in enumerate(args)] for s in (1, -1)]
        num = ((ops.layer_norm(*moved[0]).double() - ops.layer_norm(*moved[1]).double()) * dy).sum() / (2 * h)
        assert abs(num - (grads[i].double() * v).sum()) < 0.01 * (1 + (grads[i].double() * v).abs().sum() / 20)


# ---- rotary positions ------------------------------------------------------------------------------------------------------------
def turned(x, pos, f, m, interleaved, sign=1):
    """In 64 bits: the result, and the magnitude of the terms of each element."""
    r = 2 * f.numel()
    x = x.double()
    angle = (pos.double()[..., None, None] * f) * sign
    c, s = angle.cos() * m, angle.sin() * m
    a, b = (x[..., 0:r:2], x[..., 1:r:2]) if interleaved else (x[..., :r // 2], x[..., r // 2:r])
    join = (lambda u, v: torch.stack([u, v], -1).flatten(-2)) if interleaved else (lambda u, v: torch.cat([u, v], -1))
    size = join((a.abs() + b.abs()) * abs(m), (a.abs() + b.abs()) * abs(m))
    return torch.cat([join(a * c - b * s, b * c + a * s), x[..., r:]], -1), torch.cat([size, torch.zeros_like(x[..., r:])], -1)


def check_rotary(q, k, pos, f, m, interleaved):
    leaves = [t.detach().requires_grad_() for t in (q, k) if t is not None]
    outs = ops.rotary(leaves[0], leaves[1] if k is not None else None, pos, f, m, interleaved)
    outs = [o for o in outs if o is not None]
    # sine and cosine to a few steps, their angle to 2^-25 of half a turn (pi), times the magnitude, two products and a sum
    tol = 10 * U
    for x, o in zip(leaves, outs):
        want, size = turned(x.detach(), pos, f, m, interleaved)
        assert o.shape == x.shape and o.dtype == x.dtype
        within(o, want, half_step(o.dtype) * want.abs() + tol * size, "out")
        assert torch.equal(o[..., 2 * f.numel():], x[..., 2 * f.numel():])
    dys = [torch.randn(o.shape, device="cuda").to(o.dtype) for o in outs]
    for x, d, g in zip(leaves, dys, torch.autograd.grad(outs, leaves, dys)):
        want, size = turned(d, pos, f, m, interleaved, -1)
        within(g, want, half_step(g.dtype) * want.abs() + tol * size, "gradient")
    with torch.no_grad():
        assert all(torch.equal(a, b) for a, b in zip(outs, [o for o in ops.rotary(q, k, pos, f, m, interleaved) if o is not None]))


# batch, length, heads of queries and keys, head size, rotated part: the flagship's, one of everything, whole heads, odd pairs, a part that no vector fits,
# heads of many units (one token per CTA), nothing rotated, more tokens than one round of the grid
ROTARY_SHAPES = [(2, 65, 22, 2, 64, 16), (1, 1, 1, 1, 2, 2), (1, 7, 3, 1, 128, 128), (2, 5, 4, 2, 80, 20), (1, 9, 2, 2, 33, 6), (1, 3, 64, 8, 256, 256), (2, 4, 3, 1, 64, 0),
                 (3, 1500, 4, 4, 32, 32), (1, 2, 5, 0, 48, 24), (16, 1, 22, 2, 64, 16), (1, 6, 300, 300, 72, 40), (1, 200_003, 1, 1, 8, 4)]


@pytest.mark.parametrize("shape", ROTARY_SHAPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_rotary_shapes(shape, interleaved, dtype):
    B, S, H, K, D, r = shape
    gen = torch.Generator(device="cuda").manual_seed(sum(shape))
    rand = lambda *s: torch.randn(*s, device="cuda", generator=gen).to(dtype)
    pos = torch.randint(0, 1 << 20, (B, S), device="cuda", generator=gen)
    f = ops.rotary_frequencies(r, 1e4, device="cuda")[0] if r else torch.zeros(0, device="cuda", dtype=torch.float64)
    check_rotary(rand(B, S, H, D), rand(B, S, K, D) if K else None, pos, f, 1.25, interleaved)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
def test_rotary_layouts(interleaved, dtype):
    gen = torch.Generator(device="cuda").manual_seed(3)
    rand = lambda *s: torch.randn(*s, device="cuda", generator=gen).to(dtype)
    f, m = ops.rotary_frequencies(32, 1e6, dict(rope_type="yarn", factor=8.0, original_max_position_embeddings=2048), device="cuda")
    B, S, H, K, D = 2, 37, 6, 2, 64
    pos = torch.arange(S, device="cuda")
    packed = rand(B, S, H + 2 * K, D)
    check_rotary(packed[:, :, :H], packed[:, :, H:H + K], pos, f, m, interleaved)
    check_rotary(rand(B, H, S, D).transpose(1, 2), rand(B, K, S, D).transpose(1, 2), pos.int(), f, m, interleaved)
    check_rotary(rand(B, S, H, D + 1)[..., 1:], rand(B, S, K, D), pos[None], f, m, interleaved)                       # off 16 bytes
    check_rotary(rand(B, S, D, H).transpose(2, 3), rand(B, S, K, D), pos.flip(0)[None].expand(B, S), f, m, interleaved)     # columns apart
    check_rotary(rand(B, S, 1, D).expand(B, S, H, D), rand(B, 1, K, D).expand(B, S, K, D), pos - 50, f, m, interleaved)     # shared heads and tokens; before zero
    every = torch.arange(2 * S, device="cuda")[::2]
    check_rotary(rand(B, S, H, D), None, every, f[::1], m, interleaved)
    flat = rand(11, H, D)
    got, none = ops.rotary(flat, None, torch.arange(11, device="cuda"), f, m, interleaved)
    assert none is None and torch.equal(got, ops.rotary(flat[None], None, torch.arange(11, device="cuda"), f, m, interleaved)[0][0])


def test_rotary_keeps_the_layout_of_its_input():
    f = ops.rotary_frequencies(16, device="cuda")[0]
    q = torch.randn(2, 4, 9, 16, device="cuda").transpose(1, 2)
    assert ops.rotary(q, None, torch.arange(9, device="cuda"), f)[0].stride() == q.stride()


def test_rotary_gradients_of_one_side_and_of_shared_heads():
    f = ops.rotary_frequencies(16, device="cuda")[0]
    pos = torch.arange(5, device="cuda")
    q, k = (torch.randn(1, 5, h, 16, device="cuda", requires_grad=True) for h in (4, 2))
    qo, ko = ops.rotary(q, k, pos, f)
    dq, dk = torch.autograd.grad(qo.sum(), [q, k], allow_unused=True, retain_graph=True)
    want = turned(torch.ones_like(q), pos, f, 1.0, False, -1)[0]
    assert dq is not None and (dk is None or not dk.any()) and (dq - want).abs().max() < 1e-6
    dk, = torch.autograd.grad(ko.sum(), [k])
    assert (dk - want[:, :, :2]).abs().max() < 1e-6
    only, = torch.autograd.grad(ops.rotary(q.detach(), k, pos, f)[1].sum(), [k])
    assert torch.equal(only, dk)
    one = torch.randn(1, 5, 1, 16, device="cuda", requires_grad=True)
    g, = torch.autograd.grad(ops.rotary(one.expand(1, 5, 4, 16), None, pos, f)[0].sum(), [one])
    assert (g - 4 * want[:, :, :1]).abs().max() < 4e-6
    with pytest.raises(RuntimeError, match="gradient of the gradient"):
        torch.autograd.grad(ops.rotary(q, None, pos, f)[0].sum(), q, create_graph=True)


def test_rotary_edges():
    f = ops.rotary_frequencies(64, 1e4, device="cuda")[0]
    x = torch.randn(1, 2, 1, 64, device="cuda")
    assert torch.equal(ops.rotary(x, None, torch.zeros(2, device="cuda", dtype=torch.int64), f)[0], x)             # position zero turns nothing
    far = torch.tensor([(1 << 24) - 1, -(1 << 24)], device="cuda")
    want, size = turned(x, far, f, 1.0, False)
    within(ops.rotary(x, None, far, f)[0], want, (half_step(FP32) * 1 + 12 * U) * size + 1e-12, "far")
    empty = torch.zeros(2, 0, 3, 64, device="cuda")
    assert ops.rotary(empty, None, torch.zeros(0, device="cuda", dtype=torch.int64), f)[0].shape == empty.shape
    x[0, 1] = float("nan")
    out = ops.rotary(x, None, far, f)[0]
    assert out[0, 0].isfinite().all() and out[0, 1].isnan().all()


# ---- gradient norm and clipping ------------------------------------------------------------------------------------------------------
def lists():
    gen = torch.Generator(device="cuda").manual_seed(4)
    rand = lambda *s: torch.randn(*s, device="cuda", generator=gen)
    flat = rand(100_003)
    many = [rand(1 + 37 * i % 301).to((FP32, BF16, FP16)[i % 3]) for i in range(1100)]          # more than two launches hold
    return dict(one=[rand(1)], scalar=[rand(())], tail=[rand(2047), rand(2049), rand(4096)], large=[rand(3_000_001), rand(5).to(BF16)], offsets=[flat[1:70], flat[71:5000], flat[5003:]],
                mixed=[rand(129, 65), rand(64, 64).t().to(BF16), rand(0), rand(3, 5, 7).to(FP16).permute(2, 0, 1), rand(33_000).to(BF16)[1:]], many=many, none=[rand(0)],
                full=[rand(20) for _ in range(64)], over=[rand(20) for _ in range(65)])


@pytest.mark.parametrize("name", sorted(lists() if torch.cuda.is_available() else []) or ["-"])
@pytest.mark.parametrize("limit", [0.5, 1e9])
def test_clip(name, limit):
    grads = lists()[name]
    norm = math.sqrt(sum(g.double().square().sum().item() for g in grads))
    got = ops.grad_norm(grads)
    assert got.dtype == FP32 and got.shape == () and abs(got.item() - norm) <= 2 * U * norm
    factor = min(1.0, limit / (norm + 1e-6))
    out = [torch.full_like(g, 9.0) for g in grads]
    before = [g.clone() for g in grads]
    assert torch.equal(ops.clip_grad_norm(grads, limit, out=out), got)
    assert all(torch.equal(g, b) for g, b in zip(grads, before))
    # the norm, the sum, the quotient and the product: four roundings besides the result's
    for o, b in zip(out, before):
        assert o.stride() == b.stride()
        within(o, b.double() * factor, (half_step(o.dtype) + 5 * U) * (b.double() * factor).abs() + (2.0 ** -25 if o.dtype == FP16 else 0), name)
    assert torch.equal(ops.clip_grad_norm(grads, limit), got)
    assert all(torch.equal(g, o) for g, o in zip(grads, out))


def test_clip_leaves_what_is_between_alone():
    flat = torch.full((1000,), 3.0, device="cuda")
    ops.clip_grad_norm([flat[10:100], flat[101:333], flat[500:501]], 1e-3)
    touched = torch.zeros(1000, dtype=torch.bool, device="cuda")
    touched[10:100] = touched[101:333] = touched[500] = True
    assert (flat[~touched] == 3).all() and (flat[touched] < 1e-2).all()


@pytest.mark.parametrize("value,count", [(1e30, 5000), (1e-30, 5000), (3e38, 4)])
def test_clip_squares_neither_overflow_nor_vanish(value, count):
    g = torch.full((count,), value, device="cuda")
    want = g[0].double().item() * math.sqrt(count)
    norm = ops.clip_grad_norm([g], want / 4 if value > 1 else 1.0)
    if want < 3.4e38:
        assert abs(norm.item() / want - 1) < 2 * U
        if value > 1:
            assert abs(g[0].item() / (value / 4) - 1) < 1e-6
    else:
        assert norm.isinf()


def test_clip_keeps_denormal_values():
    tiny = torch.tensor([1e-40, -3e-39, 1.0, 0.0], device="cuda").repeat(700)
    grads = [tiny, tiny.to(BF16), tiny[1:]]
    out = [torch.zeros_like(g) for g in grads]
    ops.clip_grad_norm(grads, 1e9, out=out)
    assert all(torch.equal(o.view(torch.int32 if o.dtype == FP32 else torch.int16), g.view(torch.int32 if g.dtype == FP32 else torch.int16)) for o, g in zip(out, grads))


def test_clip_values_that_are_not_finite():
    for bad in (float("nan"), float("inf")):
        g, h = torch.ones(100, device="cuda"), torch.ones(5000, device="cuda", dtype=BF16)
        h[4321] = bad
        norm = ops.clip_grad_norm([g, h], 1.0)
        if bad != bad:
            assert norm.isnan() and g.isnan().all() and h.isnan().all()
        else:                                                        # the factor is zero; infinity times zero is no number
            assert norm.isinf() and not g.any() and h[4321].isnan() and not h[:4321].any()


def test_clip_refuses_and_bumps_versions():
    t, u = torch.ones(64, device="cuda"), torch.ones(64, device="cuda")
    for call in (lambda: ops.clip_grad_norm([t, t], 1.0), lambda: ops.clip_grad_norm([t, t[1:]], 1.0), lambda: ops.clip_grad_norm([t[:32], t[32:]], 1.0, out=[t[32:], t[:32]]),
                 lambda: ops.clip_grad_norm([t[:32]], 1.0, out=[t[16:48]]), lambda: ops.clip_grad_norm([t], 1.0, out=[u.to(BF16)]), lambda: ops.clip_grad_norm([t, torch.ones(3)], 1.0),
                 lambda: ops.clip_grad_norm([t.view(8, 8)[:, :4]], 1.0), lambda: ops.clip_grad_norm([t.double()], 1.0), lambda: ops.clip_grad_norm([t], 0.0)):
        with pytest.raises((RuntimeError, ValueError)):
            call()
    assert (t == 1).all()
    version = t._version
    ops.clip_grad_norm([t], 1.0)
    assert t._version > version
    w = torch.ones(64, device="cuda", requires_grad=True)
    loss = (w * u).sum()
    ops.clip_grad_norm([u], 1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    with torch.inference_mode():
        v = torch.ones(64, device="cuda")
        ops.clip_grad_norm([v], 1.0)
    assert v.norm() < 1.001


# ---- streams and graphs --------------------------------------------------------------------------------------------------------------
def test_training_ops_replay_from_a_graph_and_run_on_another_stream():
    gen = torch.Generator(device="cuda").manual_seed(12)
    rand = lambda *s: torch.randn(*s, device="cuda", generator=gen)
    f, m = ops.rotary_frequencies(64, device="cuda")
    x, w, b, pos = rand(2, 50, 4, 64), rand(64), rand(64), torch.arange(50, device="cuda")
    leaves = [t.requires_grad_() for t in (x, w, b)]

    def step():
        y = ops.layer_norm(*leaves)
        q, k = ops.rotary(y[:, :, :3], y[:, :, 3:], pos, f, m)
        grads = torch.autograd.grad([q, k], leaves, [torch.ones_like(q), torch.ones_like(k)])
        return (q, k, *grads, ops.clip_grad_norm(list(grads), 0.1))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
        other = step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for seed in (1, 2):
        with torch.no_grad():
            x.copy_(torch.randn(x.shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed)))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, e) for a, e in zip(held, step()))
    assert all(t.isfinite().all() for t in other)


def test_rotary_of_empty_heads():
    f = torch.zeros(0, device="cuda", dtype=torch.float64)
    x = torch.zeros(1, 2, 3, 0, device="cuda")
    assert ops.rotary(x, None, torch.zeros(2, device="cuda", dtype=torch.int64), f)[0].shape == x.shape
    q, k = torch.zeros(1, 2, 0, 8, device="cuda"), torch.ones(1, 2, 1, 8, device="cuda")
    qo, ko = ops.rotary(q, k, torch.zeros(2, device="cuda", dtype=torch.int64), ops.rotary_frequencies(8, device="cuda")[0])
    assert qo.shape == q.shape and torch.equal(ko, k)


@pytest.mark.parametrize("call", [
    lambda c: ops.layer_norm(c(3, 0)), lambda c: ops.layer_norm(c(3, 4, dtype=torch.float64)), lambda c: ops.layer_norm(c(3, 4), c(3)), lambda c: ops.layer_norm(c(3, 4), torch.ones(4)),
    lambda c: ops.layer_norm(c(3, 4), eps=-1.0), lambda c: ops.layer_norm(c(3, 4, dtype=BF16), out_dtype=FP32), lambda c: ops.layer_norm(c(3, 4), None, c(4, 1)),
    lambda c: ops.rotary(c(1, 2, 3, 8), None, torch.zeros(2, dtype=torch.int64), c(4, dtype=torch.float64)), lambda c: ops.rotary(c(1, 2, 3, 8), None, c(2, dtype=torch.int64), c(4)),
    lambda c: ops.rotary(c(1, 2, 3, 8), c(1, 2, 3, 6), c(2, dtype=torch.int64), c(4, dtype=torch.float64)), lambda c: ops.rotary(c(1, 2, 3, 8), None, c(3, dtype=torch.int64), c(4, dtype=torch.float64)),
    lambda c: ops.rotary(c(1, 2, 3, 8), None, c(2, dtype=torch.int64), c(5, dtype=torch.float64)), lambda c: ops.rotary(c(1, 2, 3, 8, dtype=torch.float64), None, c(2, dtype=torch.int64), c(4, dtype=torch.float64)),
    lambda c: ops.grad_norm([]), lambda c: ops.grad_norm([c(3, dtype=torch.int64)]),
])
def test_refusals_on_the_gpu(call):
    with pytest.raises(ValueError):
        call(lambda *shape, **kw: torch.zeros(*shape, device="cuda", **kw))


def test_operators_in_two_threads():
    """Calls at once from two threads, on a stream each."""
    import threading
    x, g = torch.randn(512, 640, device="cuda"), [torch.randn(3000, device="cuda") for _ in range(70)]
    f = ops.rotary_frequencies(64, device="cuda")[0]
    pos, results = torch.arange(512, device="cuda"), {}
    torch.cuda.synchronize()

    def work(who):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                leaf = x.clone().requires_grad_()
                y = ops.layer_norm(leaf)
                q, _ = ops.rotary(y.view(512, 10, 64), None, pos, f)
                d, = torch.autograd.grad(q, leaf, torch.ones_like(q))
                results[who] = (q.detach(), d, ops.clip_grad_norm(g, 1.0, out=[torch.empty_like(t) for t in g]))
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert all(torch.equal(a, b) for a, b in zip(results[0], results[1]))


# ---- more elements than 32 bits count ---------------------------------------------------------------------------------------------------
def test_layer_norm_of_more_than_2_31_elements():
    rows, dim = 2_100_000, 1032
    x = torch.randn(4096, dim, device="cuda").to(BF16).repeat(rows // 4096 + 1, 1)[:rows].requires_grad_()
    w = torch.randn(dim, device="cuda")
    y = ops.layer_norm(x, w)
    dx, = torch.autograd.grad(y, x, y.detach())
    tail = x.detach()[-7:].clone().requires_grad_()
    y7 = ops.layer_norm(tail, w)
    assert torch.equal(y[-7:], y7) and torch.equal(dx[-7:], torch.autograd.grad(y7, tail, y7.detach())[0])


def test_rotary_of_more_than_2_31_elements():
    f = ops.rotary_frequencies(256, device="cuda")[0]
    tokens = 2_200_000
    q = torch.randn(1, 4096, 4, 256, device="cuda").to(BF16).repeat(1, tokens // 4096 + 1, 1, 1)[:, :tokens]
    pos = torch.arange(tokens, device="cuda")
    out = ops.rotary(q, None, pos, f)[0]
    assert torch.equal(out[:, -9:], ops.rotary(q[:, -9:], None, pos[-9:], f)[0])


def test_clip_of_more_than_2_31_elements():
    n = 2 ** 31 + 77
    g = torch.full((n,), 2.0 ** -10, device="cuda", dtype=BF16)
    g[-3:] = 1.0
    norm = ops.clip_grad_norm([g], 1.0)
    want = math.sqrt((n - 3) * 2.0 ** -20 + 3)
    assert abs(norm.item() / want - 1) <= 2 * U
    scaled = torch.tensor([2.0 ** -10 / want, 1 / want]).to(BF16).tolist()
    assert g[0].item() == g[n // 2].item() == g[-4].item() == scaled[0] and g[-3:].tolist() == [scaled[1]] * 3
