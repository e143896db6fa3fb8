"""GPU: layer norm with its gradients, AdamW over many tensors and the 8-bit product against plain statements of the same
operators in float64 on the CPU.

Tolerances count roundings: u = 2^-24 is half a step of fp32; a sum of n terms in fp32 is off by at most (longest chain of
additions) * u * (sum of magnitudes).  A row's sums pass at most 32 additions in a lane, 6 in a wave, 4 over waves and
some more for longer rows: 64 is above all of them for H <= 20000.  A 16-bit result adds one rounding of its own."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
U = 2.0 ** -24
DT = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


@pytest.fixture(scope="module")
def ops():
    from stdiff_amd import ops as _ops
    return _ops


def rnd(*shape, seed=0, scale=1.0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale


def half_step(t):
    return torch.finfo(t.dtype).eps / 2 if t.dtype != torch.float32 else U


def within(got, want, tol, what):
    got, want = got.detach().cpu().double(), want.double()
    assert got.shape == want.shape
    off = (got - want).abs() - tol
    assert bool((off <= 0).all()), f"{what}: off by up to {float(off.max()):.3e} more than the tolerance"


# ---------------------------------------------------------------- layer norm
SIZES = [(1, 1), (1, 7), (3, 64), (5, 257), (130, 512), (2, 513), (7, 1001), (9, 1024), (3, 1025), (4, 2048), (3, 2051), (2, 4096),
         (3, 4099), (2, 8192), (3, 8193), (2, 20000), (70, 65), (40, 129), (33, 300), (2, 16384), (2, 16385)]
KINDS = [("fp32", "fp32", "fp32"), ("fp32", "bf16", "fp32"), ("bf16", "bf16", "fp32"), ("bf16", "fp32", "bf16"), ("fp16", "fp16", "fp16"),
         ("fp32", "fp16", "fp16")]


def norm64(x, w, b, eps):
    x = x.double()
    mean = x.mean(1, keepdim=True)
    rstd = 1 / torch.sqrt(((x - mean) ** 2).mean(1, keepdim=True) + eps)
    y = (x - mean) * rstd
    if w is not None:
        y = y * w.double()
    return (y if b is None else y + b.double()), mean, rstd


def norm_tol(x, w, b, mean, rstd):
    """(x - mean) is off by 65 u of the row's magnitudes, rstd by 130 u of itself / 2, two products and a sum follow"""
    x = x.double()
    size = (x.abs() + x.abs().mean(1, keepdim=True) + (x - mean).abs()) * rstd
    size = size * (1 if w is None else w.double().abs())
    return 70 * U * size + U * (0 if b is None else b.double().abs()) + 1e-12


@pytest.mark.parametrize("R,H", SIZES)
@pytest.mark.parametrize("xt,yt,wt", KINDS)
def test_layer_norm(ops, R, H, xt, yt, wt):
    x = (rnd(R, H, seed=1) * 2 + rnd(R, 1, seed=2, scale=3.0)).to(DT[xt])
    w, b = (1 + rnd(H, seed=3, scale=0.2)).to(DT[wt]), rnd(H, seed=4).to(DT[wt])
    mean, rstd = torch.empty(R, device=DEV), torch.empty(R, device=DEV)
    y = ops.layer_norm(x.to(DEV), w.to(DEV), b.to(DEV), eps=1e-5, out_dtype=DT[yt], mean=mean, rstd=rstd)
    want, m64, r64 = norm64(x, w, b, 1e-5)
    assert y.dtype == DT[yt]
    within(y, want, norm_tol(x, w, b, m64, r64) * 1.01 + half_step(y) * want.abs() * 1.01, "y")
    within(mean.view(-1, 1), m64, 65 * U * x.double().abs().mean(1, keepdim=True) + U * m64.abs(), "mean")
    # relative error of rstd: half of the variance's; the variance of a row of one element is zero
    within(rstd.view(-1, 1), r64, 70 * U * r64 + r64 ** 3 * 65 * U * x.double().abs().mean(1, keepdim=True) ** 2, "rstd")


def test_layer_norm_without_parameters_and_strides(ops):
    big = rnd(6, 300, seed=5).to(DEV)
    x = big[::2, 3:260]                                       # rows 600 apart, first element at 12 bytes
    for w, b in ((None, None), (rnd(257, seed=6), None), (None, rnd(257, seed=7))):
        out = torch.full((3, 400), 7.0, device=DEV)
        got = ops.layer_norm(x, None if w is None else w.to(DEV), None if b is None else b.to(DEV), out=out[:, 1:258])
        assert got.data_ptr() == out[:, 1:258].data_ptr()
        want, m, r = norm64(x.cpu(), w, b, 1e-6)
        within(got, want, norm_tol(x.cpu(), w, b, m, r) + U * want.abs(), "strided")
        assert bool((out[:, 0] == 7).all()) and bool((out[:, 258:] == 7).all())
    one = rnd(1, 96, seed=8).to(DEV)
    wide = ops.layer_norm(one.expand(5, 96))                  # one row for all
    assert torch.equal(wide, ops.layer_norm(one).expand(5, 96))
    for H in (96, 3000, 9000):
        x = rnd(3, H, seed=9).to(DEV)
        want = ops.layer_norm(x, eps=1e-6)
        assert torch.equal(ops.layer_norm(x, out=x), want) and torch.equal(x, want)
    assert ops.layer_norm(torch.empty(0, 64, device=DEV)).shape == (0, 64)


def test_layer_norm_far_mean_and_special_rows(ops):
    x = rnd(4, 1024, seed=10) + torch.tensor([[0.0], [1e4], [0.0], [0.0]])
    x[2] = 3.25                                                # no spread: y is the bias
    x[3, 17] = float("nan")
    b = rnd(1024, seed=11)
    y = ops.layer_norm(x.to(DEV), None, b.to(DEV)).cpu()
    want, m, r = norm64(x, None, b, 1e-6)
    # row 1: the mean's own error (65 u * 1e4) moves all elements alike, the spread keeps its digits
    within(y[:3], want[:3], norm_tol(x, None, b, m, r)[:3] + U * want[:3].abs(), "far mean")
    assert torch.equal(y[2], b) and bool(torch.isnan(y[3]).all()) and bool(torch.isfinite(y[:3]).all())


GRAD_KINDS = [("fp32", "fp32", "fp32"), ("fp32", "bf16", "fp32"), ("bf16", "bf16", "bf16"), ("fp16", "fp16", "fp32"), ("bf16", "fp32", "fp32")]


def grad64(dy, x, mean, rstd, w):
    dy, x, mean, rstd = dy.double(), x.double(), mean.double().view(-1, 1), rstd.double().view(-1, 1)
    hat = (x - mean) * rstd
    g = dy if w is None else dy * w.double()
    dx = rstd * (g - g.mean(1, keepdim=True) - hat * (g * hat).mean(1, keepdim=True))
    return dx, (dy * hat).sum(0), dy.sum(0), hat, g


def grad_tol(dy, rstd, hat, g):
    """dx: sums of at most 65 additions over products of 3 roundings; columns: a chain of the rows of a wave and the joins"""
    dy, rstd = dy.double(), rstd.double().view(-1, 1)
    dx = rstd * (4 * g.abs() + 70 * g.abs().mean(1, keepdim=True) + 76 * hat.abs() * (g * hat).abs().mean(1, keepdim=True)) * U
    chain = dy.shape[0] / 64 + 64
    return dx + 1e-14, (chain + 4) * U * (dy * hat).abs().sum(0) + 1e-14, chain * U * dy.abs().sum(0) + 1e-14


@pytest.mark.parametrize("R,H", SIZES + [(700, 320), (1500, 320), (2077, 1001), (40, 9001), (2500, 64), (2100, 1024), (2300, 2051), (2060, 4099), (2200, 8192), (1030, 100), (1026, 9000)])
@pytest.mark.parametrize("xt,dt,wt", GRAD_KINDS)
def test_layer_norm_bwd(ops, R, H, xt, dt, wt):
    x = (rnd(R, H, seed=20) + rnd(R, 1, seed=21)).to(DT[xt])
    dy, w = rnd(R, H, seed=22, scale=0.1).to(DT[dt]), (1 + rnd(H, seed=23, scale=0.2)).to(DT[wt])
    _, mean, rstd = norm64(x, None, None, 1e-5)
    mean, rstd = mean.view(-1).float(), rstd.view(-1).float()
    dx, dw, db = ops.layer_norm_bwd(dy.to(DEV), x.to(DEV), mean.to(DEV), rstd.to(DEV), w.to(DEV))
    wx, ww, wb, hat, g = grad64(dy, x, mean, rstd, w)
    tx, tw, tb = grad_tol(dy, rstd, hat, g)
    assert dx.dtype == x.dtype and dw.dtype == db.dtype == torch.float32
    within(dx, wx, tx * 1.01 + half_step(dx) * wx.abs() * 1.01 + (2.0 ** -25 if xt == "fp16" else 0), "dx")   # fp16: half of its last step
    within(dw, ww, tw, "dweight")
    within(db, wb, tb, "dbias")


@pytest.mark.parametrize("R,H", [(37, 48), (37, 1024), (37, 3000), (37, 8200), (5000, 48), (2500, 1024)])
def test_layer_norm_bwd_options(ops, R, H):
    big, bigdy = rnd(R, H + 5, seed=30).to(DEV), rnd(R, H + 3, seed=31).to(DEV)
    x, dy, w = big[:, 2:H + 2], bigdy[:, 1:H + 1], rnd(H, seed=32).to(DEV)
    mean, rstd = torch.empty(R, device=DEV), torch.empty(R, device=DEV)
    ops.layer_norm(x, w, mean=mean, rstd=rstd)
    dx, dw, db = ops.layer_norm_bwd(dy, x, mean, rstd, w)
    # the formulas' own statistics: against differences of the forward, in float64
    wx, ww, wb, hat, g = grad64(dy.cpu(), x.cpu(), mean.cpu(), rstd.cpu(), w.cpu())
    tx, tw, tb = grad_tol(dy.cpu(), rstd.cpu(), hat, g)
    within(dx, wx, tx + U * wx.abs(), "strided dx")
    again = ops.layer_norm_bwd(dy, x, mean, rstd, w)
    assert all(torch.equal(p, q) for p, q in zip((dx, dw, db), again))           # a fixed order of additions
    # accumulate, only one of the two, and none
    dw2, db2 = dw.clone(), db.clone()
    ops.layer_norm_bwd(dy, x, mean, rstd, w, dweight=dw2, dbias=db2, accumulate=True)
    assert torch.equal(dw2, dw + dw) and torch.equal(db2, db + db)
    only = torch.empty(H, device=DEV)
    r = ops.layer_norm_bwd(dy, x, mean, rstd, None, dbias=only)
    assert r[1] is None and torch.equal(only, db)
    plain = ops.layer_norm_bwd(dy, x, mean, rstd)
    assert plain[1] is None and plain[2] is None
    within(plain[0], grad64(dy.cpu(), x.cpu(), mean.cpu(), rstd.cpu(), None)[0], grad_tol(dy.cpu(), rstd.cpu(), hat, dy.cpu().double())[0] + U, "no weight")
    # in place of dy and of x, with a workspace of its own
    ws = torch.full((ops.layer_norm_bwd_workspace(R, H, torch.float32),), float("nan"), device=DEV)
    for which in ("dy", "x"):
        a, c = dy.clone(), x.clone()
        got = ops.layer_norm_bwd(a, c, mean, rstd, w, dx=a if which == "dy" else c, workspace=ws)
        assert torch.equal(got[0], dx) and torch.equal(got[1], dw) and torch.equal(got[2], db)
    # one gradient row for all rows, as the backward of a sum gives it
    row = rnd(1, H, seed=33).to(DEV)
    a = ops.layer_norm_bwd(row.expand(R, H), x, mean, rstd, w)
    b = ops.layer_norm_bwd(row.expand(R, H).contiguous(), x, mean, rstd, w)
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    e = torch.empty(0, H, device=DEV)
    z = torch.empty(0, device=DEV)
    r = ops.layer_norm_bwd(e, e, z, z, w)
    assert r[0].shape == (0, H) and float(r[1].abs().sum()) == 0 and float(r[2].abs().sum()) == 0


def test_layer_norm_gradient_against_differences(ops):
    """d(sum(c * y)) by x, w and b: central differences of the forward in float64 against the kernel's gradients."""
    R, H, h = 3, 20, 1e-5
    x, c = rnd(R, H, seed=40).double(), rnd(R, H, seed=41).double()
    w, b = rnd(H, seed=42).double(), rnd(H, seed=43).double()
    mean, rstd = torch.empty(R, device=DEV), torch.empty(R, device=DEV)
    ops.layer_norm(x.float().to(DEV), w.float().to(DEV), b.float().to(DEV), mean=mean, rstd=rstd)
    got = ops.layer_norm_bwd(c.float().to(DEV), x.float().to(DEV), mean, rstd, w.float().to(DEV))

    def f(x_, w_, b_):
        return float((norm64(x_, w_, b_, 1e-6)[0] * c).sum())
    args = [x, w, b]
    for k in range(3):
        d = torch.zeros_like(args[k])
        for i in range(d.numel()):
            e = torch.zeros_like(d).view(-1)
            e[i] = h
            e = e.view_as(d)
            d.view(-1)[i] = (f(*[a + e if j == k else a for j, a in enumerate(args)]) - f(*[a - e if j == k else a for j, a in enumerate(args)])) / (2 * h)
        # h^2 times a third derivative of order 100, and float32 inputs: far below 1e-4
        assert float((got[k].cpu().double() - d).abs().max()) < 1e-4 * max(1.0, float(d.abs().max())), k


# ---------------------------------------------------------------- AdamW
def blocks_of(x):
    n = x.numel()
    k = -(-n // 256)
    out = torch.zeros(k * 256, dtype=x.dtype)
    out[:n] = x.reshape(-1)
    return out.view(k, 256)


def code8(x, root):
    """e4m3 codes and scales of a tensor as the operator defines them, in float32 operation by operation"""
    b = blocks_of(x)
    top = b.abs().amax(1, keepdim=True)
    top = torch.where(top > 0, top.clamp_min(1e-30), top)
    f = torch.where(top > 0, torch.full_like(top, 448.0) / top, torch.zeros_like(top))
    z = b * f
    if root:
        z = torch.where(b > 0, z.clamp_min(2.0 ** -9), z)
    return z.to(torch.float8_e4m3fn).view(-1)[:x.numel()], (top / torch.full_like(top, 448.0)).view(-1)


def held8(code, scale):
    return code.float().reshape(-1) * scale.repeat_interleave(256)[:code.numel()]


class Oracle:
    """the state and step of one tensor, states held in float32 (or 8 bits), arithmetic in `dt`"""

    def __init__(self, p, bits, wd, dt):
        self.p, self.bits, self.wd, self.dt = p.clone(), bits, wd, dt
        n = p.numel()
        self.m, self.v = torch.zeros(n), torch.zeros(n)
        if bits == 8:
            self.m, self.ms = code8(self.m, False)
            self.v, self.vs = code8(self.v, True)

    def step(self, g, t, lr, coef, b1, b2, eps):
        dt = self.dt
        g = (g.reshape(-1).to(dt) * torch.tensor(coef, dtype=dt))
        if self.bits == 8:
            m, r = held8(self.m, self.ms).to(dt), held8(self.v, self.vs).to(dt)
            v = r * r
        else:
            m, v = self.m.to(dt), self.v.to(dt)
        m = m * b1 + g * (1 - b1)
        v = v * b2 + g * g * (1 - b2)
        # by way of float64: torch's float32 square root on the CPU is not the correctly rounded one on every host, and the
        # root of a float32 rounded to float64 and then to float32 is (53 >= 2 * 24 + 2 bits)
        root = torch.sqrt(v.double()).to(dt)
        one = torch.ones((), dtype=dt)
        den = root / (one * math.sqrt(1 - b2 ** t)) + eps
        p = self.p.reshape(-1).to(dt)
        p = p * (one - lr * (one * self.wd)) - (one * (lr / (1 - b1 ** t))) * (m / den)
        self.p = p.to(self.p.dtype).view(self.p.shape)
        self.raw = m, root
        if self.bits == 8:
            self.m, self.ms = code8(m.float(), False)
            self.v, self.vs = code8(root.float(), True)
        else:
            self.m, self.v = m.float(), v.float()


LENGTHS = [(1,), (3,), (255,), (256,), (257,), (64, 64), (0,), (4096,), (4097,), (333, 77), (5, 4099)]


def make(ops, shapes, bits, pt, wd, seed=0):
    ps = [rnd(*s, seed=seed + i, scale=0.1).to(DT[pt]) for i, s in enumerate(shapes)]
    dp = [p.to(DEV) for p in ps]
    if bits == 8:
        st = [ops.adamw8_state(p) for p in dp]
        args = ops.adamw_multi_args(dp, [s[0] for s in st], [s[1] for s in st], [s[2] for s in st], [s[3] for s in st], weight_decay=wd)
    else:
        st = [(torch.zeros_like(p, dtype=torch.float32), torch.zeros_like(p, dtype=torch.float32)) for p in dp]
        args = ops.adamw_multi_args(dp, [s[0] for s in st], [s[1] for s in st], weight_decay=wd)
    return ps, dp, st, args


def gradients(shapes, gt, seed, scale=1e-2):
    out = []
    for i, s in enumerate(shapes):
        g = rnd(*s, seed=seed + i, scale=scale * 10 ** (i % 3 - 1))
        g.view(-1)[::7] = 0                                       # elements whose gradient is exactly zero
        if i % 4 == 3:
            g[:] = 0                                              # a whole tensor without one
        out.append(g.to(DT[gt]))
    return out


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("pt,gt", [("fp32", "fp32"), ("fp32", "bf16"), ("bf16", "bf16"), ("fp16", "fp32")])
def test_adamw_multi_steps(ops, bits, pt, gt):
    """Several steps without clipping: states bit for bit what the formulas give operation by operation in float32 (the codes
    and scales of 8 bits among them), parameters against the same step in float64."""
    wd = [0.1 if len(s) == 2 else 0.0 for s in LENGTHS]
    ps, dp, st, args = make(ops, LENGTHS, bits, pt, wd)
    same = [Oracle(p, bits, w, torch.float32) for p, w in zip(ps, wd)]
    step = torch.zeros(1, device=DEV, dtype=torch.int32)
    lr, b1, b2, eps = 1e-3, 0.9, 0.999, 1e-8
    for t in range(1, 6):
        gs = gradients(LENGTHS, gt, 100 * t)
        before = [p.cpu().clone() for p in dp]
        ops.adamw_multi(args, [g.to(DEV) for g in gs], step, lr, betas=(b1, b2), eps=eps)
        assert int(step) == t
        for i, (o, g) in enumerate(zip(same, gs)):
            o.p = before[i]
            exact = Oracle(before[i].double(), bits, wd[i], torch.float64)
            exact.m, exact.v = o.m, o.v
            if bits == 8:
                exact.ms, exact.vs = o.ms, o.vs
            exact.step(g, t, lr, 1.0, b1, b2, eps)
            o.step(g, t, lr, 1.0, b1, b2, eps)
            m, v = st[i][0].cpu().view(-1), st[i][1].cpu().view(-1)
            if bits == 8:
                assert torch.equal(m.view(torch.uint8), o.m.view(torch.uint8)) and torch.equal(v.view(torch.uint8), o.v.view(torch.uint8)), (t, i)
                assert torch.equal(st[i][2].cpu(), o.ms) and torch.equal(st[i][3].cpu(), o.vs), (t, i)
                # against the unrounded state: half a step of e4m3, or half of its smallest step where that is more
                for code, scale, raw in ((m, o.ms, exact.raw[0]), (v, o.vs, exact.raw[1])):
                    s = scale.double().repeat_interleave(256)[:raw.numel()]
                    least = 2.0 ** -9 if code is v else 2.0 ** -10
                    within(held8(code, scale), raw, raw.abs() * (2.0 ** -4 + 1e-6) + s * least * 1.001, f"state of tensor {i}")
            else:
                assert torch.equal(m, o.m) and torch.equal(v, o.v), (t, i)
            # p: the decayed value and the step, each a handful of roundings
            upd = (exact.p.view(-1) - before[i].double().view(-1)).abs() + wd[i] * lr * before[i].double().view(-1).abs() + 2 * lr
            within(dp[i].view(-1), exact.p.view(-1), 12 * U * upd + (2 * U + half_step(dp[i])) * exact.p.view(-1).abs() * 1.001 +
                   (2.0 ** -25 if pt == "fp16" else 0), f"parameter {i}")


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_multi_clips_by_the_norm_of_all(ops, bits):
    shapes = [(257, 33), (0,), (5000,), (3,)]
    gs = gradients(shapes, "fp32", 7, scale=1.0)
    total = math.sqrt(sum(float((g.double() ** 2).sum()) for g in gs))
    for max_norm, scale in ((1.0, 1.0), (0.5 * total, 1.0), (2 * total, 1.0), (1.0, 0.125), (None, 0.25)):
        ps, dp, st, args = make(ops, shapes, bits, "fp32", 0.0)
        step, norm = torch.zeros(1, device=DEV, dtype=torch.int32), torch.zeros(1, device=DEV)
        ops.adamw_multi(args, [g.to(DEV) for g in gs], step, 1e-3, max_norm=max_norm, grad_scale=scale, norm=norm)
        assert abs(float(norm) - total * scale) < 100 * U * total * scale
        coef = scale * (1.0 if max_norm is None else min(1.0, max_norm / (total * scale + 1e-6)))
        for i, g in enumerate(gs):
            o = Oracle(ps[i].double(), bits, 0.0, torch.float64)
            o.step(g, 1, 1e-3, coef, 0.9, 0.999, 1e-8)
            within(dp[i], o.p, 300 * U * 1e-3 + 3 * U * o.p.abs(), "p")
            if bits == 32:
                within(st[i][0].view(-1), o.m, 110 * U * o.m.double().abs(), "m")
                within(st[i][1].view(-1), o.v, 220 * U * o.v.double().abs(), "v")


def test_adamw_multi_more_tensors_than_one_table(ops):
    """over a hundred tensors, tiny and large ones mixed: the same as each of them alone; a None gradient changes nothing"""
    shapes = [(i % 9 * 37 + 1,) if i % 10 else (90, 130) for i in range(125)]
    gs = gradients(shapes, "fp32", 500)
    for bits in (32, 8):
        ps, dp, st, args = make(ops, shapes, bits, "fp32", 0.01)
        step = torch.full((1,), 3, device=DEV, dtype=torch.int32)
        dg = [g.to(DEV) if i not in (4, 60, 124) else None for i, g in enumerate(gs)]
        ops.adamw_multi(args, dg, step, 1e-3, norm=torch.zeros(1, device=DEV))
        assert int(step) == 4
        for i in range(len(shapes)):
            if dg[i] is None:
                assert torch.equal(dp[i].cpu(), ps[i]) and not bool(st[i][0].cpu().view(torch.uint8).any())
                continue
            p1, d1, s1, a1 = make(ops, [shapes[i]], bits, "fp32", 0.01, seed=i)
            ops.adamw_multi(a1, [dg[i]], torch.full((1,), 3, device=DEV, dtype=torch.int32), 1e-3)
            assert torch.equal(d1[0], dp[i]) and all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(s1[0], st[i])), i
    ops.adamw_multi(args, dg, step, 1e-3)                         # and the next call takes the gradient back up
    ops.adamw_multi(args, [g.to(DEV) for g in gs], step, 1e-3)
    assert not torch.equal(dp[4].cpu(), ps[4])


def test_adamw_multi_unaligned_views(ops):
    """parameters, gradients and states that begin at any element of larger buffers; nothing beside them is touched"""
    sizes, at = [1000, 1, 513, 4099], [1, 1003, 1007, 1522]
    for bits in (32, 8):
        flat = {k: rnd(6000, seed=60 + i, scale=0.1).to(DEV) for i, k in enumerate("pg")}
        if bits == 8:
            flat["m"], flat["v"] = (torch.zeros(6000, device=DEV, dtype=torch.uint8).view(torch.float8_e4m3fn) for _ in range(2))
        else:
            flat["m"], flat["v"] = torch.zeros(6000, device=DEV), torch.zeros(6000, device=DEV)
        was = {k: v.clone() for k, v in flat.items()}
        view = {k: [v[a:a + n] for a, n in zip(at, sizes)] for k, v in flat.items()}
        sc = [[torch.zeros(-(-n // 256), device=DEV) for n in sizes] for _ in range(2)] if bits == 8 else [None, None]
        args = ops.adamw_multi_args(view["p"], view["m"], view["v"], *sc)
        ops.adamw_multi(args, view["g"], torch.zeros(1, device=DEV, dtype=torch.int32), 1e-3, max_norm=1.0)
        aligned = [t.clone() for t in [was["p"][a:a + n] for a, n in zip(at, sizes)]]
        st = [ops.adamw8_state(t) if bits == 8 else (torch.zeros_like(t), torch.zeros_like(t)) for t in aligned]
        a2 = ops.adamw_multi_args(aligned, *[[s[k] for s in st] for k in range(4 if bits == 8 else 2)])
        ops.adamw_multi(a2, [t.clone() for t in view["g"]], torch.zeros(1, device=DEV, dtype=torch.int32), 1e-3, max_norm=1.0)
        outside = torch.ones(6000, dtype=torch.bool)
        for i, (a, n) in enumerate(zip(at, sizes)):
            outside[a:a + n] = False
            assert torch.equal(view["p"][i], aligned[i])
            assert torch.equal(view["m"][i].view(torch.uint8), st[i][0].view(torch.uint8))
        for k in "pmv":
            raw = lambda t: t.view(torch.uint8).view(6000, -1)[outside.to(DEV)]  # noqa: E731
            assert torch.equal(raw(flat[k]), raw(was[k])), k


def test_adamw8_extremes(ops):
    """blocks whose elements span the whole range, tiny and huge gradients, a block without any, one with a NaN"""
    n = 256 * 6
    g = torch.zeros(n)
    g[:256] = 10.0 ** torch.linspace(-18, 2, 256)                 # far below the smallest code beside the largest
    g[256:512] = 1e-38
    g[512:768] = 3e18
    g[1024:1280] = rnd(256, seed=70)
    g[1100] = float("nan")
    g[1280:] = rnd(256, seed=71)
    p = torch.ones(n, device=DEV)
    m, v, ms, vs = ops.adamw8_state(p)
    args = ops.adamw_multi_args([p], [m], [v], [ms], [vs])
    step = torch.zeros(1, device=DEV, dtype=torch.int32)
    for _ in range(3):
        ops.adamw_multi(args, [g.to(DEV)], step, 1e-2)
        q = p.cpu()
        fine = torch.ones(n, dtype=torch.bool)
        fine[1024:1280] = False
        assert bool(torch.isfinite(q[fine]).all())
        # the step of an element is at most lr * sqrt(1 / (1 - b2)) at the very worst; no element may run away through a
        # root that was rounded to zero
        assert float((q[fine] - 1).abs().max()) < 3 * 1e-2 * 32
    assert torch.equal(p.cpu()[768:1024], torch.ones(256))        # no gradient: nothing moved
    assert bool(torch.isnan(p.cpu()[1024:1280]).all())            # the NaN took its block, and no other
    codes = v.cpu().float()
    assert bool((codes[:256] > 0).all()) and bool((codes[768:1024] == 0).all())


# ---------------------------------------------------------------- 8-bit product
@pytest.mark.parametrize("R,K", [(1, 1), (1, 15), (3, 16), (5, 1000), (2, 1024), (7, 2049), (33, 4096), (2, 9000), (0, 32)])
@pytest.mark.parametrize("xt", ["fp32", "bf16", "fp16"])
def test_quantize_rows(ops, R, K, xt):
    x = (rnd(R, K, seed=80) * torch.exp(rnd(R, 1, seed=81))).to(DT[xt])
    if R > 2:
        x[1] = 0
        x[2, ::3] = 0
    q, s = ops.quantize_rows(x.to(DEV))
    f = x.float()
    top = f.abs().amax(1, keepdim=True) if R else f[:, :1]
    want = torch.round(f * torch.where(top > 0, torch.full_like(top, 127.0) / top, torch.zeros_like(top)))
    assert q.shape == (R, K) and torch.equal(q.cpu().float(), want)
    assert torch.equal(s.cpu(), (top / torch.full_like(top, 127.0)).view(-1))
    if R:
        rows = torch.as_strided(q, (R, -(-K // 16) * 16), (q.stride(0) if R > 1 else -(-K // 16) * 16, 1))
        assert not bool(rows[:, K:].any())
        # half a step of the scale, and the roundings of the product and the scale
        within(q.cpu().float() * s.cpu().view(-1, 1), f, s.cpu().double().view(-1, 1) * (0.5 + 200 * U) + 2 * U * f.double().abs(), "value")


def test_quantize_rows_special(ops):
    x = rnd(6, 40, seed=82)
    x[0] *= 1e-37
    x[1, 3] = float("inf")
    x[2, 5] = float("nan")
    x[3] *= 1e37
    x[4] = 0
    big = torch.zeros(6, 50, device=DEV)
    big[:, 3:43] = x.to(DEV)
    out = torch.full((6, 64), 9, device=DEV, dtype=torch.int8)
    q, s = ops.quantize_rows(big[:, 3:43], out=out[:, :40])
    assert q.data_ptr() == out.data_ptr() and bool((out[:, 48:] == 9).all()) and bool((out[:, 40:48] == 0).all())
    s = s.cpu()
    assert math.isinf(float(s[1])) and math.isnan(float(s[2])) and float(s[4]) == 0 and not bool(q[4].any())
    ok = [0, 3, 5]
    within(q.cpu().float()[ok] * s[ok].view(-1, 1), x[ok], s[ok].double().view(-1, 1) * 0.501, "value")
    y = ops.gemm_i8(q, s.to(DEV), *ops.quantize_rows(rnd(8, 40, seed=83).to(DEV))).cpu()
    assert not bool(torch.isfinite(y[1:3]).any()) and bool(torch.isfinite(y[ok]).all()) and not bool(y[4].any())


def operands(M, N, K, seed=0, lo=-127, hi=128):
    g = torch.Generator().manual_seed(seed)
    kp = -(-K // 16) * 16
    A = torch.randint(lo, hi, (M, kp), generator=g, dtype=torch.int8)      # behind K: anything at all
    W = torch.randint(lo, hi, (N, kp), generator=g, dtype=torch.int8)
    return A, W, torch.rand(M, generator=g) * 0.01, torch.rand(N, generator=g) * 0.01, torch.randn(N, generator=g)


SHAPES8 = [(1, 1, 1), (1, 64, 64), (3, 5, 17), (16, 16, 64), (17, 100, 130), (128, 128, 128), (129, 127, 915), (4, 4096, 1024), (1, 1000, 2048),
           (33, 65, 4096), (300, 1000, 200), (257, 513, 1040), (64, 200, 8192), (700, 900, 64), (31, 4100, 48), (1030, 770, 333)]


@pytest.mark.parametrize("M,N,K", SHAPES8)
@pytest.mark.parametrize("ct", ["fp32", "bf16", "fp16"])
def test_gemm_i8(ops, M, N, K, ct):
    A, W, sa, sw, b = operands(M, N, K, seed=M + N + K)
    exact = (A[:, :K].double() @ W[:, :K].double().T)
    for bias in (b, None):
        y = ops.gemm_i8(A.to(DEV)[:, :K], sa.to(DEV), W.to(DEV)[:, :K], sw.to(DEV), None if bias is None else bias.to(DEV), out_dtype=DT[ct])
        prod = exact * sa.double().view(-1, 1) * sw.double()
        want = prod if bias is None else prod + bias.double()
        assert y.dtype == DT[ct]
        within(y, want, 4 * U * (prod.abs() + want.abs()) + half_step(y) * want.abs() * 1.001 + (2.0 ** -25 if ct == "fp16" else 0), "y")


@pytest.mark.parametrize("M,N", [(1600, 1700), (2600, 2500), (3300, 2900), (5000, 4200)])
@pytest.mark.parametrize("K", [33, 128, 200, 384, 915, 1040])
def test_gemm_i8_large_outputs(ops, M, N, K):
    """sizes of the tiled kernels: 128 x 128 tiles; 256 x 256 tiles cut in halves, whole ones, and more than there are CUs with
    a last round in halves; one slab of K, two, three and many, whole and cut.  What lies beside C is left alone."""
    A, W, sa, sw, b = [t.to(DEV) for t in operands(M, N, K, seed=M + K)]
    prod = A[:, :K].double() @ W[:, :K].double().t().contiguous() * sa.double().view(-1, 1) * sw.double()
    want = prod + b.double()
    tol = 4 * U * (prod.abs() + want.abs())
    for ct in (torch.float32, torch.bfloat16):
        out = torch.full((M + 1, N + 8), 5.0, device=DEV, dtype=ct)
        y = ops.gemm_i8(A[:, :K], sa, W[:, :K], sw, b, out=out[:M, 3:3 + N])
        off = (y.double() - want).abs() - tol - half_step(y) * want.abs() * 1.001
        assert float(off.max()) <= 0, (ct, float(off.max()))
        assert bool((out[:, :3] == 5).all()) and bool((out[:, 3 + N:] == 5).all()) and bool((out[M] == 5).all())
        again = ops.gemm_i8(A[:, :K], sa, W[:, :K], sw, b, out_dtype=ct)
        assert torch.equal(again, y)


@pytest.mark.parametrize("M,N,K", [(2, 3, 131071), (200, 300, 131071), (600, 1024, 2048), (1500, 1300, 1000)])
def test_gemm_i8_sum_is_exact(ops, M, N, K):
    """the largest sums that can be: all operands at -128 / 127; with scales of one, C is the rounded whole number"""
    A, W, _, _, _ = operands(M, N, K, seed=5, lo=-128, hi=128)
    A[0], W[0], A[-1] = -128, -128, 127
    one_m, one_n = torch.ones(M, device=DEV), torch.ones(N, device=DEV)
    y = ops.gemm_i8(A.to(DEV)[:, :K], one_m, W.to(DEV)[:, :K], one_n).cpu()
    rows, cols = torch.tensor([0, M // 2, M - 1]), torch.tensor([0, N // 2, N - 1])
    want = (A[rows][:, :K].long() @ W[cols][:, :K].long().T)
    assert torch.equal(y[rows][:, cols], want.float())
    if K < 10000:
        assert torch.equal(y, (A[:, :K].double() @ W[:, :K].double().T).float())


def test_gemm_i8_strides_and_edges(ops):
    """row strides of all operands larger than their rows, an output that begins anywhere; what lies beside is left alone"""
    for M, N, K in ((5, 7, 33), (130, 250, 300), (520, 1031, 200)):
        A, W, sa, sw, b = operands(M, N, K, seed=9)
        bigA = torch.full((M, 1024), 77, device=DEV, dtype=torch.int8)
        bigW = torch.full((N, 512), -99, device=DEV, dtype=torch.int8)
        bigA[:, 48:48 + K], bigW[:, 16:16 + K] = A[:, :K].to(DEV), W[:, :K].to(DEV)
        want = ops.gemm_i8(A.to(DEV)[:, :K], sa.to(DEV), W.to(DEV)[:, :K], sw.to(DEV), b.to(DEV), out_dtype=torch.bfloat16)
        for dt in (torch.bfloat16, torch.float32):
            out = torch.full((M, N + 9), 3.0, device=DEV, dtype=dt)
            got = ops.gemm_i8(bigA[:, 48:48 + K], sa.to(DEV), bigW[:, 16:16 + K], sw.to(DEV), b.to(DEV), out=out[:, 5:5 + N])
            assert torch.equal(got.bfloat16(), want)
            assert bool((out[:, :5] == 3).all()) and bool((out[:, 5 + N:] == 3).all())
    z = ops.gemm_i8(torch.empty(0, 16, device=DEV, dtype=torch.int8), torch.empty(0, device=DEV), W.to(DEV)[:, :16], sw.to(DEV))
    assert z.shape == (0, N)


# ---------------------------------------------------------------- sizes whose offsets pass 32 bits
def test_far_rows(ops):
    """rows behind the 2^32-th byte (and the 2^31-th element): the same results as the same rows alone"""
    H, ld = 1001, 40000
    R = 2 ** 31 // ld + 100                                     # the last rows begin behind element 2^31
    far = torch.zeros(R, ld, device=DEV, dtype=torch.bfloat16)
    last = rnd(50, H, seed=110).to(DEV).bfloat16()
    far[-50:, 7:7 + H] = last
    x = far[:, 7:7 + H]
    w, b = rnd(H, seed=111).to(DEV), rnd(H, seed=112).to(DEV)
    mean, rstd = torch.empty(R, device=DEV), torch.empty(R, device=DEV)
    assert torch.equal(ops.layer_norm(x, w, b, mean=mean, rstd=rstd)[-50:], ops.layer_norm(last, w, b))
    dx, dw, db = ops.layer_norm_bwd(x, x, mean, rstd, w)
    one = ops.layer_norm_bwd(last, last, mean[-50:].clone(), rstd[-50:].clone(), w)
    assert torch.equal(dx[-50:], one[0])
    scale = last.float().pow(2).sum(0) * float(rstd.max()) + 1
    assert bool(((dw - one[1]).abs() <= 200 * U * scale).all())   # the other rows add zeros: another order of the same terms
    q, s = ops.quantize_rows(x)
    q1, s1 = ops.quantize_rows(last)
    assert torch.equal(q[-50:], q1) and torch.equal(s[-50:], s1)
    del x, far, dx, q
    M, K, N = 2 ** 31 // 8192 + 300, 8192, 300
    A = torch.zeros(M, K, device=DEV, dtype=torch.int8)
    A[-300:] = torch.randint(-127, 128, (300, K), device=DEV, dtype=torch.int8)
    W = torch.randint(-127, 128, (N, K), device=DEV, dtype=torch.int8)
    sa, sw = torch.rand(M, device=DEV), torch.rand(N, device=DEV)
    y = ops.gemm_i8(A, sa, W, sw)
    assert torch.equal(y[-300:], ops.gemm_i8(A[-300:], sa[-300:].clone(), W, sw)) and not bool(y[:-300].any())


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_multi_far_elements(ops, bits):
    """a tensor of more than 2^31 elements: its ends as small tensors of their own give them"""
    n = 2 ** 31 + 5000
    p, g = torch.zeros(n, device=DEV, dtype=torch.bfloat16), torch.zeros(n, device=DEV, dtype=torch.bfloat16)
    cut = 2 ** 31 - 2048
    p[cut:], g[cut:] = rnd(n - cut, seed=120).to(DEV).bfloat16(), rnd(n - cut, seed=121).to(DEV).bfloat16()
    small = p[cut:].clone()
    if bits == 8:
        st, own = ops.adamw8_state(p), ops.adamw8_state(small)
    else:
        st, own = [tuple(torch.zeros(t.numel(), device=DEV) for _ in range(2)) for t in (p, small)]
    step = torch.zeros(2, device=DEV, dtype=torch.int32)
    for t, s, gr, k in ((p, st, g, 0), (small, own, g[cut:].clone(), 1)):
        args = ops.adamw_multi_args([t], *[[v] for v in s])
        ops.adamw_multi(args, [gr], step[k:k + 1], 1e-2)
    assert torch.equal(p[cut:], small) and not bool(p[:cut].any())
    assert torch.equal(st[0][cut:].view(torch.uint8), own[0].view(torch.uint8))
    assert torch.equal(st[1][cut:].view(torch.uint8), own[1].view(torch.uint8))


# ---------------------------------------------------------------- refusals
def test_refusals(ops):
    x, w = torch.zeros(4, 32, device=DEV), torch.ones(32, device=DEV)
    s4, s32 = torch.zeros(4, device=DEV), torch.zeros(32, device=DEV)
    with pytest.raises(ValueError, match="neighbours"):
        ops.layer_norm(x.t())
    with pytest.raises(ValueError, match="weight"):
        ops.layer_norm(x, w[:31])
    with pytest.raises(TypeError):
        ops.layer_norm(x, w, w.bfloat16())
    with pytest.raises(TypeError):
        ops.layer_norm(x.half(), w.bfloat16())
    with pytest.raises(TypeError):
        ops.layer_norm(x.double())
    with pytest.raises(ValueError, match="overlap"):
        ops.layer_norm(x, out=torch.zeros(32, device=DEV).expand(4, 32))
    with pytest.raises(ValueError):
        ops.layer_norm(x, eps=-1.0)
    with pytest.raises(ValueError, match="mean"):
        ops.layer_norm_bwd(x, x, None, None)
    with pytest.raises(ValueError, match="accumulate"):
        ops.layer_norm_bwd(x, x, s4, s4, w, accumulate=True)
    many, s9 = torch.zeros(9000, 32, device=DEV), torch.zeros(9000, device=DEV)
    with pytest.raises(ValueError, match="workspace"):
        ops.layer_norm_bwd(many, many, s9, s9, w, workspace=torch.zeros(4, device=DEV))
    with pytest.raises(ValueError, match="dy"):
        ops.layer_norm_bwd(x[:3], x, s4, s4, w)
    with pytest.raises(TypeError):
        ops.layer_norm_bwd(x, x, s4, s4, w, dx=x.bfloat16())
    p, m, v = (torch.zeros(300, device=DEV) for _ in range(3))
    args = ops.adamw_multi_args([p], [m], [v])
    step = torch.zeros(1, device=DEV, dtype=torch.int32)
    for bad in ([p[:299]], [p.cpu()], [torch.zeros(600, device=DEV)[::2]], [p, p], []):
        with pytest.raises(ValueError):
            ops.adamw_multi(args, bad, step, 1e-3)
    with pytest.raises(TypeError):
        ops.adamw_multi(args, [p.double()], step, 1e-3)
    for kw in (dict(max_norm=0.0), dict(max_norm=float("nan")), dict(betas=(1.0, 0.9)), dict(eps=-1.0), dict(workspace=torch.zeros(3, device=DEV))):
        with pytest.raises(ValueError):
            ops.adamw_multi(args, [p], step, 1e-3, **kw)
    with pytest.raises(ValueError):
        ops.adamw_multi(args, [p], step, -1e-3)
    with pytest.raises(ValueError):
        ops.adamw_multi(args, [p], step.long(), 1e-3)
    assert int(step) == 0 and not bool(p.any())
    with pytest.raises(TypeError):
        ops.adamw_multi_args([p], [m.half()], [v])
    with pytest.raises(ValueError):
        ops.adamw_multi_args([p], [m[:7]], [v])
    with pytest.raises(ValueError, match="share"):
        ops.adamw_multi_args([p, p], [m, torch.zeros_like(m)], [v, torch.zeros_like(v)])
    with pytest.raises(ValueError, match="share"):
        ops.adamw_multi_args([p], [m], [m])
    with pytest.raises(ValueError, match="share"):
        ops.adamw_multi_args([p[:200], p[199:]], [m[:200], torch.zeros(101, device=DEV)], [v[:200], torch.zeros(101, device=DEV)])
    moved = torch.nn.Parameter(torch.zeros(300, device=DEV))
    margs = ops.adamw_multi_args([moved], [m], [v])
    moved.data = torch.ones(300, device=DEV)
    with pytest.raises(ValueError, match="memory"):
        ops.adamw_multi(margs, [p], step, 1e-3)
    c, c2 = m.to(torch.float8_e4m3fn), m.to(torch.float8_e4m3fn)
    with pytest.raises(ValueError):
        ops.adamw_multi_args([p], [c], [c2])
    with pytest.raises(ValueError):
        ops.adamw_multi_args([p], [c], [c2], [torch.zeros(1, device=DEV)], [torch.zeros(2, device=DEV)])
    q = torch.zeros(4, 32, device=DEV, dtype=torch.int8)
    with pytest.raises(TypeError, match="int8"):
        ops.gemm_i8(x, s4, q, s4)
    with pytest.raises(ValueError, match="borders"):
        ops.gemm_i8(q[:, 3:], s4, q[:, 3:], s4)
    with pytest.raises(ValueError, match="borders"):
        ops.gemm_i8(torch.zeros(4, 33, device=DEV, dtype=torch.int8), s4, q, s4)
    with pytest.raises(ValueError, match="borders"):                 # the last row ends with its memory
        ops.gemm_i8(torch.zeros(3 * 48 + 33, device=DEV, dtype=torch.int8).as_strided((4, 33), (48, 1)), s4, q, s4)
    with pytest.raises(ValueError, match="columns"):
        ops.gemm_i8(q, s4, q[:, :16], s4)
    with pytest.raises(ValueError, match="a_scale"):
        ops.gemm_i8(q, s32, q, s4)
    with pytest.raises(ValueError):
        ops.gemm_i8(*[torch.zeros(1, 131072, device=DEV, dtype=torch.int8), s4[:1]] * 2)
    with pytest.raises(TypeError):
        ops.gemm_i8(q, s4, q, s4, out_dtype=torch.float64)
    with pytest.raises(ValueError, match="borders"):
        ops.quantize_rows(x[:, :30], out=torch.zeros(4, 30, device=DEV, dtype=torch.int8))


# ---------------------------------------------------------------- together, as they are used
@pytest.mark.parametrize("bits", [32, 8])
def test_projection_is_trained_and_served(ops, bits):
    """LayerNorm -> Linear: forward, backward and AdamW on all four tensors for a few steps against autograd and the same
    optimizer in float64; then the matrix in 8 bits, served one token and many at a time."""
    R, H, N, lr = 200, 96, 64, 1e-2
    x, target = rnd(R, H, seed=90) * 2 + 1, rnd(R, N, seed=91)
    shapes = [(H,), (H,), (N, H), (N,)]
    init = [torch.ones(H), torch.zeros(H), rnd(N, H, seed=92, scale=0.1), torch.zeros(N)]
    dp = [p.to(DEV) for p in init]
    if bits == 8:
        st = [ops.adamw8_state(p) for p in dp]
    else:
        st = [(torch.zeros_like(p), torch.zeros_like(p)) for p in dp]
    args = ops.adamw_multi_args(dp, *[[s[k] for s in st] for k in range(len(st[0]))], weight_decay=[0, 0, 0.1, 0])
    step = torch.zeros(1, device=DEV, dtype=torch.int32)
    oracles = [Oracle(p.double(), bits, w, torch.float64) for p, w in zip(init, (0, 0, 0.1, 0))]
    mean, rstd = torch.empty(R, device=DEV), torch.empty(R, device=DEV)
    dx_, dt_ = x.to(DEV), target.to(DEV)
    for t in range(1, 4):
        y = ops.layer_norm(dx_, dp[0], dp[1], mean=mean, rstd=rstd)
        d = (y @ dp[2].t() + dp[3] - dt_) * (2.0 / (R * N))
        _, dw, db = ops.layer_norm_bwd(d @ dp[2], dx_, mean, rstd, dp[0])
        grads = [dw, db, d.t().contiguous() @ y, d.sum(0)]
        leaves = [o.p.clone().requires_grad_() for o in oracles]
        out = norm64(x, leaves[0], leaves[1], 1e-6)[0] @ leaves[2].T + leaves[3]
        ((out - target.double()) ** 2).mean().backward()
        for g, l in zip(grads, leaves):
            assert float((g.cpu().double() - l.grad).abs().max()) < 1e-4 * float(l.grad.abs().max())
        total = math.sqrt(sum(float((l.grad ** 2).sum()) for l in leaves))
        norm = torch.zeros(1, device=DEV)
        ops.adamw_multi(args, grads, step, lr, max_norm=0.1, norm=norm)
        assert abs(float(norm) - total) < 1e-5 * total
        for o, l in zip(oracles, leaves):
            o.step(l.grad, t, lr, min(1.0, 0.1 / (total + 1e-6)), 0.9, 0.999, 1e-8)
        for p, o in zip(dp, oracles):
            # float32 gradients 1e-6 apart; in 8 bits a state next to a border may fall to the other code, an eighth of a
            # moment at most, for a few elements
            off = (p.cpu().double() - o.p).abs()
            assert float(off.max()) < (0.2 if bits == 8 else 2e-3) * lr * t and float(off.median()) < 1e-4 * lr
    wq, ws = ops.quantize_rows(dp[2])
    for rows in (1, R):
        y = ops.layer_norm(dx_[:rows], dp[0], dp[1], out_dtype=torch.bfloat16)
        served = ops.gemm_i8(*ops.quantize_rows(y), wq, ws, dp[3], out_dtype=torch.bfloat16)
        yf, wf = y.cpu().double(), dp[2].cpu().double()
        want = yf @ wf.T + dp[3].cpu().double()
        # each operand is off by half of its step: sum over K of (|y| sw + |w| sy) / 2 + sy sw / 4 is above the error
        sy, sw = yf.abs().amax(1, keepdim=True) / 127, wf.abs().amax(1) / 127
        tol = (yf.abs().sum(1, keepdim=True) * sw + sy * wf.abs().sum(1)) * 0.501 + H * sy * sw * 0.251 + want.abs() * 2.0 ** -8
        within(served, want, tol, "served")


@pytest.mark.parametrize("bits", [32, 8])
def test_model_is_trained_by_adamw_multi(ops, bits):
    """The framework's denoiser through its autograd path, its parameters (condi_emb has no gradient) updated by adamw_multi:
    states as the formulas give them from the same gradients, and a forward that sees the new weights."""
    from stdiff_amd.model.stDiff_model import DiT_stDiff
    torch.manual_seed(3)
    C_, G, H = 24, 40, 128
    model = DiT_stDiff(G, H, 1, "dit", 4, 6).to(DEV)
    with torch.no_grad():
        for p in model.parameters():
            p.add_(0.02 * torch.randn_like(p))                  # the output and adaLN layers begin with zeros
    params = list(model.parameters())
    decay = [0.01 if p.dim() == 2 else 0.0 for p in params]
    if bits == 8:
        st = [ops.adamw8_state(p) for p in params]
    else:
        st = [(torch.zeros_like(p), torch.zeros_like(p)) for p in params]
    x, y, t = rnd(C_, G, seed=1).to(DEV), rnd(C_, G, seed=2).to(DEV), torch.arange(C_, device=DEV)
    states = [[s[k] for s in st] for k in range(len(st[0]))]
    early = ops.adamw_multi_args(params, *states, weight_decay=decay)
    model(x, t, y)                                              # the autograd path gathers the parameters in one buffer
    step, norm = torch.zeros(1, device=DEV, dtype=torch.int32), torch.zeros(1, device=DEV)
    with pytest.raises(ValueError, match="memory"):
        ops.adamw_multi(early, [None] * len(params), step, 1e-2)
    args = ops.adamw_multi_args(params, *states, weight_decay=decay)
    own = [Oracle(p.detach().cpu(), bits, w, torch.float32) for p, w in zip(params, decay)]
    for k in range(1, 4):
        for p in params:
            p.grad = None
        before = model(x, t, y)
        (before ** 2).mean().backward()
        grads = [p.grad for p in params]
        assert sum(g is None for g in grads) == 1
        was = [p.detach().cpu().clone() for p in params]
        ops.adamw_multi(args, grads, step, 1e-2, norm=norm)
        total = math.sqrt(sum(float((g.double() ** 2).sum()) for g in grads if g is not None))
        assert abs(float(norm) - total) < 100 * U * total
        for p, o, g, w, s in zip(params, own, grads, was, st):
            if g is None:
                assert torch.equal(p.detach().cpu(), w)
                continue
            o.p = w
            o.step(g.cpu(), k, 1e-2, 1.0, 0.9, 0.999, 1e-8)
            assert torch.equal(s[0].cpu().view(-1).view(torch.uint8), o.m.view(torch.uint8))
            assert torch.equal(s[1].cpu().view(-1).view(torch.uint8), o.v.view(torch.uint8))
            within(p, o.p, 16 * U * 3e-2 + 3 * U * o.p.double().abs(), "parameter")
        fresh = DiT_stDiff(G, H, 1, "dit", 4, 6).to(DEV)
        fresh.load_state_dict(model.state_dict())
        with torch.no_grad():
            assert torch.equal(model(x, t, y), fresh(x, t, y)) and not torch.equal(model(x, t, y), before)


def test_captured_step_replays(ops):
    """layer_norm, its backward and the optimizer in one ops.Graph with workspaces of their own, the program's own eager work
    between the replays: every replay gives what the eager calls give on the same data."""
    R, H = 70, 200
    ws = [torch.empty(ops.layer_norm_bwd_workspace(R, H, torch.float32), device=DEV), torch.empty(ops.adamw_multi_workspace(2), device=DEV)]
    x, dy = torch.empty(R, H, device=DEV), torch.empty(R, H, device=DEV)
    y, dx = torch.empty_like(x), torch.empty_like(x)
    mean, rstd, dw, db, norm = (torch.empty(n, device=DEV) for n in (R, R, H, H, 1))
    q, qs = torch.empty(R, 208, device=DEV, dtype=torch.int8)[:, :H], torch.empty(R, device=DEV)
    out = torch.empty(R, R, device=DEV)
    for bits in (32, 8):
        ps, dp, st, args = make(ops, [(H,), (H,)], bits, "fp32", 0.01)
        ps2, dp2, st2, args2 = make(ops, [(H,), (H,)], bits, "fp32", 0.01)
        step, step2 = (torch.zeros(1, device=DEV, dtype=torch.int32) for _ in range(2))

        def body():
            ops.layer_norm(x, dp[0], dp[1], out=y, mean=mean, rstd=rstd)
            ops.layer_norm_bwd(dy, x, mean, rstd, dp[0], dx=dx, dweight=dw, dbias=db, workspace=ws[0])
            ops.adamw_multi(args, [dw, db], step, 1e-2, max_norm=1.0, norm=norm, workspace=ws[1])
            ops.quantize_rows(y, out=q, scale=qs)
            ops.gemm_i8(q, qs, q, qs, out=out)
        g = ops.Graph()
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            g.begin()
            body()
            g.end()
        torch.cuda.synchronize()
        assert int(step) == 0
        for k in range(4):
            x.copy_(rnd(R, H, seed=200 + k).to(DEV))
            dy.copy_(rnd(R, H, seed=300 + k).to(DEV))
            with torch.cuda.stream(s):
                s.wait_stream(torch.cuda.default_stream())
                g.launch()
            torch.cuda.synchronize()
            m2, r2 = torch.empty(R, device=DEV), torch.empty(R, device=DEV)
            y2 = ops.layer_norm(x, dp2[0], dp2[1], mean=m2, rstd=r2)
            dx2, dw2, db2 = ops.layer_norm_bwd(dy, x, m2, r2, dp2[0])
            ops.adamw_multi(args2, [dw2, db2], step2, 1e-2, max_norm=1.0)
            q2, qs2 = ops.quantize_rows(y2)
            out2 = ops.gemm_i8(q2, qs2, q2, qs2)
            for a, b in ((y, y2), (dx, dx2), (dw, dw2), (db, db2), (dp[0], dp2[0]), (dp[1], dp2[1]), (out, out2), (qs, qs2)):
                assert torch.equal(a, b), (bits, k)
            assert int(step) == int(step2) == k + 1


def test_side_stream(ops):
    """calls enqueue on the stream that is current, and on no other"""
    x = rnd(512, 1024, seed=95).to(DEV)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        ops.spin_probe(1, 2000)
        x.mul_(2)                                                # done after the wait; the calls below have to see it
        y = ops.layer_norm(x)
        q, sc = ops.quantize_rows(x)
        z = ops.gemm_i8(q, sc, q, sc)
    s.synchronize()
    assert torch.equal(y, ops.layer_norm(x)) and torch.equal(q, ops.quantize_rows(x)[0]) and torch.equal(z, ops.gemm_i8(q, sc, q, sc))


@pytest.mark.parametrize("H", [3, 48, 100, 320, 1000, 1024, 2051, 9001, 17000])
@pytest.mark.parametrize("xt", ["fp32", "bf16"])
def test_layer_norm_in_place_and_beside(ops, H, xt):
    """out in x's place, and out and x as columns of one buffer: the bits of a call with memory of its own"""
    R = 70
    x, w, b = rnd(R, H, seed=400).to(DT[xt]).to(DEV), rnd(H, seed=401).to(DEV), rnd(H, seed=402).to(DEV)
    want = ops.layer_norm(x, w, b)
    buf = torch.full((R, 3 * H + 5), 7.0, device=DEV, dtype=DT[xt])
    a, out = buf[:, 1:H + 1], buf[:, H + 1:2 * H + 1]
    a.copy_(x)
    assert ops.layer_norm(a, w, b, out=out) is out and torch.equal(out, want) and torch.equal(a, x)
    ops.layer_norm(a, w, b, out=a)
    assert torch.equal(a, want) and torch.equal(out, want)
    assert bool((buf[:, :1] == 7).all()) and bool((buf[:, 2 * H + 1:] == 7).all())


def test_gemm_i8_very_many_columns(ops):
    """more columns than a launch of 16 each can have; the first and the last ones are right, the gap behind them stays"""
    N, K = (1 << 27) + 40, 16
    W = torch.zeros(N, K, device=DEV, dtype=torch.int8)
    at = torch.tensor([0, 1, 77, 1 << 26, (1 << 26) + 13, (1 << 27) - 1, 1 << 27, N - 17, N - 1], device=DEV)
    rows = torch.randint(-127, 128, (len(at), K), generator=torch.Generator().manual_seed(5)).to(torch.int8)
    W[at] = rows.to(DEV)
    A = torch.randint(-127, 128, (1, K), generator=torch.Generator().manual_seed(6)).to(torch.int8)
    sa, sw = torch.full((1,), 0.5, device=DEV), torch.full((N,), 0.25, device=DEV)
    C = torch.full((1, N + 8), 9.0, device=DEV)
    ops.gemm_i8(A.to(DEV), sa, W, sw, out=C[:, :N])
    want = (A.long() @ rows.long().t()).double()[0] * 0.125
    assert torch.equal(C[0, at].cpu().double(), want)
    assert bool((C[0, N:] == 9).all())
    C[0, at] = 0
    assert not bool(C[0, :N].any())


def test_two_threads(ops):
    """calls of two threads on streams of their own, with other sizes and types: each gets what it gets alone"""
    import threading
    jobs = [(300, 1000, torch.float32, 1e-2), (257, 520, torch.bfloat16, 3e-2)]

    def work(k, n):
        R, H, t, lr = jobs[k]
        x, dy = rnd(R, H, seed=410 + k).to(t).to(DEV), rnd(R, H, seed=420 + k).to(t).to(DEV)
        p = torch.ones(H, device=DEV)
        m, v = torch.zeros_like(p), torch.zeros_like(p)
        args, step = ops.adamw_multi_args([p], [m], [v]), torch.zeros(1, device=DEV, dtype=torch.int32)
        mean, rstd = torch.empty(R, device=DEV), torch.empty(R, device=DEV)
        for _ in range(n):
            y = ops.layer_norm(x, p, mean=mean, rstd=rstd)
            dx, dw, db = ops.layer_norm_bwd(dy, x, mean, rstd, p)
            ops.adamw_multi(args, [dw], step, lr, max_norm=1.0)
            q, s = ops.quantize_rows(y)
            z = ops.gemm_i8(q, s, q, s)
        torch.cuda.current_stream().synchronize()
        return p, dx, z
    alone = [work(k, 30) for k in range(2)]
    together, failed = [None, None], []

    def thread(k):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                together[k] = work(k, 30)
        except BaseException as e:
            failed.append(e)
    torch.cuda.synchronize()
    ts = [threading.Thread(target=thread, args=(k,)) for k in range(2)]
    for t in ts:
        t.start()
    for t in ts:
        t.join()
    assert not failed
    for k in range(2):
        for a, b in zip(alone[k], together[k]):
            assert torch.equal(a, b), k


def test_torch_graph(ops):
    """the same calls with outputs and workspaces of their own allocation, captured by torch.cuda.graph"""
    R, H = 2200, 260
    x, dy, w = torch.empty(R, H, device=DEV), torch.empty(R, H, device=DEV), rnd(H, seed=430).to(DEV)
    mean, rstd = torch.empty(R, device=DEV), torch.empty(R, device=DEV)

    def body(mean, rstd):
        y = ops.layer_norm(x, w, mean=mean, rstd=rstd)
        q, s = ops.quantize_rows(y)
        return (y, s, ops.gemm_i8(q, s, q[:100], s[:100])) + ops.layer_norm_bwd(dy, x, mean, rstd, w)
    x.zero_(), dy.zero_()
    body(mean, rstd)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = body(mean, rstd)
    for k in range(4):
        x.copy_(rnd(R, H, seed=440 + k).to(DEV))
        dy.copy_(rnd(R, H, seed=450 + k).to(DEV))
        g.replay()
        want = body(torch.empty_like(mean), torch.empty_like(rstd))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b), k


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_multi_edges(ops, bits):
    """no tensors, no gradients, empty tensors, a norm that nothing is clipped by, the largest and smallest clips"""
    step, norm = torch.zeros(1, device=DEV, dtype=torch.int32), torch.full((1,), 5.0, device=DEV)
    none = ops.adamw_multi_args([], [], [])
    ops.adamw_multi(none, [], step, 1e-2, max_norm=1.0, norm=norm)
    assert int(step) == 1 and float(norm) == 0
    ps, dp, st, args = make(ops, [(300,), (0,), (5,)], bits, "fp32", 0.1)
    before = [p.clone() for p in dp]
    norm.fill_(5)
    ops.adamw_multi(args, [None, None, None], step, 1e-2, max_norm=1.0, norm=norm)
    assert int(step) == 2 and float(norm) == 0 and all(torch.equal(a, b) for a, b in zip(dp, before))
    gs = [torch.full((300,), 2.0, device=DEV), torch.empty(0, device=DEV), None]
    step.zero_()
    ops.adamw_multi(args, gs, step, 0.0, norm=norm)                  # lr 0: the states move, the parameters stay
    assert abs(float(norm) - 1200 ** 0.5) < 1e-3 and all(torch.equal(a, b) for a, b in zip(dp, before))
    m = st[0][0].float() * (st[0][2].repeat_interleave(256)[:300] if bits == 8 else 1)
    assert bool((abs(m - 0.2) < 1e-6).all())
    step.zero_()
    for max_norm, grad_scale in ((1e-45, 1.0), (1e300, 1.0), (1.0, 1e-30)):
        ops.adamw_multi(args, gs, step, 1e-3, max_norm=max_norm, grad_scale=grad_scale)
    assert all(bool(torch.isfinite(p).all()) for p in dp) and torch.equal(dp[2], before[2])


def test_written_tensors_and_moved_states(ops):
    """what a call wrote counts as changed for autograd; states that were given other memory are refused"""
    x = rnd(9, 32, seed=460).to(DEV)
    w = torch.ones(32, device=DEV)
    mean, rstd, sc = (torch.ones(9, device=DEV) for _ in range(3))
    q, out = torch.empty(9, 32, device=DEV, dtype=torch.int8), torch.empty(9, 9, device=DEV)
    dw, db, dx = torch.zeros(32, device=DEV), torch.zeros(32, device=DEV), torch.empty_like(x)
    a = torch.ones(9, 32, device=DEV, requires_grad=True)
    b = a * x                                                        # saves x
    for call, changed in ((lambda: ops.layer_norm_bwd(x, x, mean, rstd, w, dx=dx, dweight=dw, dbias=db), (dx, dw, db)),
                          (lambda: ops.quantize_rows(x, out=q, scale=sc), (q, sc)), (lambda: ops.gemm_i8(q, sc, q, sc, out=out), (out,)),
                          (lambda: ops.layer_norm(x, out=x, mean=mean, rstd=rstd), (x, mean, rstd))):
        before = [t._version for t in changed]
        call()
        assert all(t._version > v for t, v in zip(changed, before))
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        b.sum().backward()
    with torch.inference_mode():
        y = torch.ones(3, 32, device=DEV)
        ops.layer_norm(y, out=y)
    assert not bool(y.any())
    p, m, v = (torch.zeros(300, device=DEV) for _ in range(3))
    args, step = ops.adamw_multi_args([p], [m], [v]), torch.zeros(1, device=DEV, dtype=torch.int32)
    ops.adamw_multi(args, [torch.ones(300, device=DEV)], step, 1e-3)
    v.data = torch.zeros(300, device=DEV)
    with pytest.raises(ValueError, match="memory"):
        ops.adamw_multi(args, [torch.ones(300, device=DEV)], step, 1e-3)
    assert int(step) == 1


@pytest.mark.parametrize("M,N", [(8192, 6400), (8000, 6500)])
@pytest.mark.parametrize("K", [128, 256, 300, 640, 1024])
def test_gemm_i8_many_tiles_per_workgroup(ops, M, N, K):
    """a workgroup's tiles follow one another with loads and stores of the last one under way: whole tiles behind whole and cut ones, one to
    eight slabs, both types of C, the same bits every time"""
    A, W, sa, sw, b = [t.to(DEV) for t in operands(M, N, K, seed=M + K)]
    prod = A[:, :K].double() @ W[:, :K].double().t().contiguous()
    prod *= sa.double().view(-1, 1)
    prod *= sw.double()
    for ct in (torch.float32, torch.bfloat16):
        for bias in (b, None):
            want = prod + bias.double() if bias is not None else prod
            y = ops.gemm_i8(A[:, :K], sa, W[:, :K], sw, bias, out_dtype=ct)
            off = (y.double() - want).abs() - 4 * U * (prod.abs() + want.abs()) - half_step(y) * want.abs() * 1.001
            assert float(off.max()) <= 0, (ct, float(off.max()))
            for _ in range(8):
                assert torch.equal(ops.gemm_i8(A[:, :K], sa, W[:, :K], sw, bias, out_dtype=ct), y)


@pytest.mark.parametrize("xt", ["fp32", "bf16"])
@pytest.mark.parametrize("R,K", [(1000, 3), (999, 64), (1001, 100), (517, 128), (515, 129), (1003, 300), (301, 512), (300, 513), (90000, 1000), (3, 1025), (70, 2048), (45000, 2100)])
def test_quantize_rows_groups_of_lanes(ops, R, K, xt):
    """rows that share a wave, rows of a workgroup, and more than a cache holds: q and scale as the formula has them, padding zero"""
    x = torch.randn(R, K, device=DEV, generator=torch.Generator(DEV).manual_seed(R + K)).to(DT[xt])
    x[R // 2] = 0
    q, s = ops.quantize_rows(x)
    top = x.float().abs().amax(1, keepdim=True)
    want = torch.round(x.float() * torch.where(top > 0, torch.full_like(top, 127.0) / top, torch.zeros_like(top)))
    assert torch.equal(s, (top / torch.full_like(top, 127.0)).view(-1)) and torch.equal(q.float(), want)
    kp = -(-K // 16) * 16
    assert not bool(torch.as_strided(q, (R, kp), (kp, 1))[:, K:].any())


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_multi_keeps_apart(ops, bits):
    """gradients, step_dev, norm and a given workspace share no memory with parameters and states, norm, step_dev and workspace none
    with the gradients or each other; nothing is changed by a call that is refused"""
    buf = rnd(8192, seed=470).to(DEV)
    p = [buf[:300], buf[1024:2024], buf[600:900]]
    free = [buf[300:600], buf[2024:3024], buf[4096:4396]]
    if bits == 8:
        st = [ops.adamw8_state(t) for t in p]
        scales = [[s[k] for s in st] for k in (2, 3)]
    else:
        st = [(buf[5000:5300], buf[5300:5600]), (torch.zeros_like(p[1]), torch.zeros_like(p[1])), (torch.zeros_like(p[2]), torch.zeros_like(p[2]))]
        buf[5300:5600].zero_()
        scales = [None, None]
    args = ops.adamw_multi_args(p, [s[0] for s in st], [s[1] for s in st], *scales)
    step, norm = torch.zeros(1, device=DEV, dtype=torch.int32), torch.zeros(1, device=DEV)
    ws = torch.empty(ops.adamw_multi_workspace(3), device=DEV)
    before, states = buf.clone(), [[t.clone() for t in s] for s in st]

    def refused(match, grads=free, step=step, **kw):
        with pytest.raises(ValueError, match=match):
            ops.adamw_multi(args, grads, step, 1e-3, **kw)
    last = buf.view(torch.bfloat16)[2 * 899 + 1:][:300]          # begins in the last two bytes of a parameter
    for i, bad in ((0, buf[299:599]), (0, buf[301:601]), (0, p[0]), (1, buf[100:1100]), (1, buf[1500:2500]), (2, buf[700:1000]), (2, last)):
        refused(f"gradient {i} shares memory", [bad if k == i else t for k, t in enumerate(free)])
    if bits == 8:
        for k in range(2):                                       # codes and scales
            refused("gradient 2 shares memory", free[:2] + [st[1][k].view(torch.uint8).view(torch.bfloat16)[100:400]])
            refused("norm shares memory", norm=st[1][2 + k][1:2])
    else:
        refused("gradient 0 shares memory", [buf[5299:5599], free[1], free[2]])
        refused("norm shares memory", norm=buf[5599:5600])
    as_int = buf.view(torch.int32)
    refused("step_dev shares memory", step=as_int[1024:1025])
    refused("norm shares memory", norm=buf[899:900])
    refused("workspace shares memory", workspace=buf[:8192])
    refused("norm and gradient 1 share memory", norm=buf[3023:3024])
    refused("step_dev and gradient 0 share memory", step=as_int[300:301])
    refused("workspace and gradient 2 share memory", workspace=buf[4395:4999])
    refused("workspace and norm share memory", workspace=ws, norm=ws[-1:])
    refused("workspace and step_dev share memory", workspace=ws, step=ws.view(torch.int32)[:1])
    refused("norm and step_dev share memory", norm=norm, step=norm.view(torch.int32))
    for kw in (dict(max_norm=0.0), dict(max_norm=float("nan")), dict(betas=(1.0, 0.9)), dict(eps=-1.0), dict(workspace=torch.zeros(3, device=DEV))):
        refused(".", **kw)
    assert torch.equal(buf, before) and int(step) == 0
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for s, t in zip(st, states) for a, b in zip(s, t))
    # beside each other they may lie, as long as they are apart: the step of tensors of their own
    own = [t.clone() for t in p]
    so = [ops.adamw8_state(t) if bits == 8 else (torch.zeros_like(t), torch.zeros_like(t)) for t in own]
    if bits == 32:
        st[0][0].zero_()
    ops.adamw_multi(ops.adamw_multi_args(own, *[[s[k] for s in so] for k in range(len(so[0]))]), [t.clone() for t in free], step.clone(), 1e-3, max_norm=1.0)
    ops.adamw_multi(args, free, as_int[900:901].zero_(), 1e-3, max_norm=1.0, norm=buf[901:902], workspace=buf[6000:])
    assert all(torch.equal(a, b) for a, b in zip(p, own)) and int(as_int[900]) == 1 and float(buf[901]) > 0


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_multi_raises_version_counters(ops, bits):
    """everything that a step writes counts as changed for autograd, what it leaves alone does not"""
    p = [torch.ones(300, device=DEV), torch.ones(40, device=DEV), torch.ones(0, device=DEV)]
    st = [ops.adamw8_state(t) if bits == 8 else (torch.zeros_like(t), torch.zeros_like(t)) for t in p]
    args = ops.adamw_multi_args(p, *[[s[k] for s in st] for k in range(len(st[0]))])
    step, norm = torch.zeros(1, device=DEV, dtype=torch.int32), torch.zeros(1, device=DEV)
    x = torch.ones(300, device=DEV, requires_grad=True)
    saved = x * st[0][-1][:1].float()                             # saves a state
    written, left = [p[0], *st[0], step, norm], [p[1], *st[1], p[2], *st[2]]
    before = [[t._version for t in ts] for ts in (written, left)]
    ops.adamw_multi(args, [torch.ones(300, device=DEV), None, torch.ones(0, device=DEV)], step, 1e-3, norm=norm)
    assert all(t._version > v for t, v in zip(written, before[0]))
    assert all(t._version == v for t, v in zip(left, before[1]))
    if bits == 8:
        assert st[0][3]._version > before[0][4]
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        saved.sum().backward()
    ops.adamw_multi(args, [None] * 3, step, 1e-3)                 # the step count alone
    assert step._version > before[0][-2] + 1
    with torch.inference_mode():                                  # tensors without counters
        q = torch.ones(8, device=DEV)
        s = [ops.adamw8_state(q)] if bits == 8 else [(torch.zeros_like(q), torch.zeros_like(q))]
        ops.adamw_multi(ops.adamw_multi_args([q], *[[t[k] for t in s] for k in range(len(s[0]))]), [torch.ones(8, device=DEV)],
                        torch.zeros(1, device=DEV, dtype=torch.int32), 1e-3)
        assert bool((q < 1).all())


@pytest.mark.parametrize("xt", ["fp32", "bf16"])
@pytest.mark.parametrize("K", [40, 300, 1000, 3000, 9000])
def test_quantize_rows_of_tiny_values(ops, xt, K):
    """rows whose largest magnitude is far below one: the formula down to 4e-37, below it the scale of 4e-37"""
    tops = torch.tensor([2e-30, 9e-31, 1e-33, 3e-35, 5e-37, 4.1e-37, 3e-37, 2e-38, 1e-39, 5e-42])
    x = rnd(len(tops), K, seed=480).clamp(-1, 1)
    x[:, 3] = -1
    x = (x * tops.view(-1, 1)).to(DT[xt])
    q, s = ops.quantize_rows(x.to(DEV))
    f = x.float()
    top = f.abs().amax(1, keepdim=True)
    top = torch.where(top > 0, top.clamp_min(4e-37), top)        # bf16 holds the last row as zeros
    assert torch.equal(s.cpu(), (top / torch.full_like(top, 127.0)).view(-1))
    assert torch.equal(q.cpu().float(), torch.round(f * torch.where(top > 0, torch.full_like(top, 127.0) / top, torch.zeros_like(top))))
    # half a step of the scale, the roundings of the product, and half of fp32's smallest step in the scale, 127 times
    within(q.cpu().double() * s.cpu().double().view(-1, 1), f, s.cpu().double().view(-1, 1) * (0.5 + 200 * U) + 2 * U * f.double().abs() + 127 * 2.0 ** -150, "value")


@pytest.mark.parametrize("R,H", [(37, 7), (37, 48), (37, 1024), (37, 3000), (37, 8200), (20, 17000), (5000, 48), (2500, 1024), (2077, 1001), (3000, 301), (2100, 4099)])
@pytest.mark.parametrize("xt", ["fp32", "bf16"])
def test_layer_norm_bwd_column_sums_of_strided_rows(ops, R, H, xt):
    """x and dy begin at odd elements, with strides of their own: dx, dweight and dbias against float64"""
    big, bigdy = rnd(R, H + 5, seed=490).to(DT[xt]).to(DEV), rnd(R, H + 3, seed=491).to(DT[xt]).to(DEV)
    x, dy, w = big[:, 3:H + 3], bigdy[:, 1:H + 1], rnd(H, seed=492).to(DEV)
    mean, rstd = torch.empty(R, device=DEV), torch.empty(R, device=DEV)
    ops.layer_norm(x, w, mean=mean, rstd=rstd)
    wx, ww, wb, hat, g = grad64(dy.cpu(), x.cpu(), mean.cpu(), rstd.cpu(), w.cpu())
    tx, tw, tb = grad_tol(dy.cpu(), rstd.cpu(), hat, g)
    dx, dw, db = ops.layer_norm_bwd(dy, x, mean, rstd, w)
    within(dx, wx, tx * 1.01 + half_step(dx) * wx.abs() * 1.01, "dx")
    within(dw, ww, tw, "dweight")
    within(db, wb, tb, "dbias")


def near(got, want, tol, what):
    """within() for tensors on the device"""
    off = (got.double() - want).abs() - tol
    assert bool((off <= 0).all()), f"{what}: off by up to {float(off.max()):.3e} more than the tolerance"


def rows_on_device(R, H, t, seed):
    gen = torch.Generator(DEV).manual_seed(seed)
    x = torch.randn(R, H, device=DEV, generator=gen)
    return (x + torch.randn(R, 1, device=DEV, generator=gen)).to(DT[t])


# calls that move more than 256 MiB: every kernel that goes past the caches (8, 32 and 64 lanes per row, the workgroup, the large workgroup
# of fp32 rows), rows that end in a cut vector among them
@pytest.mark.parametrize("R,H,xt,yt", [(400000, 127, "fp32", "fp32"), (150000, 301, "fp32", "bf16"), (50000, 1001, "fp32", "bf16"), (44000, 1024, "fp32", "bf16"),
                                       (22000, 2051, "fp32", "bf16"), (5100, 9001, "fp32", "bf16"), (1000000, 72, "bf16", "bf16"), (250000, 300, "bf16", "bf16"),
                                       (70000, 1001, "bf16", "bf16"), (33000, 2048, "bf16", "bf16"), (17000, 4099, "bf16", "bf16"), (7500, 9001, "fp16", "fp16")])
def test_layer_norm_past_the_caches(ops, R, H, xt, yt):
    x, w, b = rows_on_device(R, H, xt, 500), (1 + rnd(H, seed=501, scale=0.2)).to(DEV), rnd(H, seed=502).to(DEV)
    assert R * H * (x.element_size() + torch.finfo(DT[yt]).bits // 8) > 256 << 20
    mean, rstd = torch.empty(R, device=DEV), torch.empty(R, device=DEV)
    y = ops.layer_norm(x, w, b, out_dtype=DT[yt], mean=mean, rstd=rstd)
    step = (1 << 24) // H + 1
    for i in range(0, R, step):                                   # rows by rows: float64 of all of them is large
        r = slice(i, min(R, i + step))
        want, m, s = norm64(x[r], w, b, 1e-6)
        tol = norm_tol(x[r], w, b, m, s) * 1.01 + half_step(y) * want.abs() * 1.01 + (2.0 ** -25 if yt == "fp16" else 0)
        near(y[r], want, tol, "y")
        size = x[r].double().abs().mean(1, keepdim=True)
        near(mean[r].view(-1, 1), m, 65 * U * size + U * m.abs(), "mean")
        near(rstd[r].view(-1, 1), s, 70 * U * s + s ** 3 * 65 * U * size ** 2, "rstd")


@pytest.mark.parametrize("R,H,xt,dt", [(230000, 100, "fp32", "fp32"), (75000, 300, "fp32", "fp32"), (23000, 1001, "fp32", "fp32"), (22000, 1024, "fp32", "fp32"),
                                       (11000, 2051, "fp32", "fp32"), (11000, 2048, "fp32", "fp32"), (2500, 9001, "fp32", "fp32"), (700000, 72, "bf16", "bf16"),
                                       (150000, 301, "bf16", "bf16"), (45000, 1024, "bf16", "bf16"), (11000, 4099, "bf16", "bf16"), (3800, 9001, "bf16", "fp32")])
def test_layer_norm_bwd_past_the_caches(ops, R, H, xt, dt):
    x, dy, w = rows_on_device(R, H, xt, 510), rows_on_device(R, H, dt, 511), (1 + rnd(H, seed=512, scale=0.2)).to(DEV)
    assert R * H * (2 * x.element_size() + dy.element_size()) > 256 << 20
    mean, rstd = torch.empty(R, device=DEV), torch.empty(R, device=DEV)
    ops.layer_norm(x, w, mean=mean, rstd=rstd)
    dx, dw, db = ops.layer_norm_bwd(dy, x, mean, rstd, w)
    ww, wb, sw, sb = (torch.zeros(H, device=DEV, dtype=torch.float64) for _ in range(4))
    step = (1 << 24) // H + 1
    for i in range(0, R, step):
        r = slice(i, min(R, i + step))
        wx, pw, pb, hat, g = grad64(dy[r], x[r], mean[r], rstd[r], w)
        near(dx[r], wx, grad_tol(dy[r], rstd[r], hat, g)[0] * 1.01 + half_step(dx) * wx.abs() * 1.01, "dx")
        ww, wb, sw, sb = ww + pw, wb + pb, sw + (dy[r].double() * hat).abs().sum(0), sb + dy[r].double().abs().sum(0)
    # grad_tol's bound over all rows: chains of the rows of a wave and the joins
    near(dw, ww, (R / 64 + 68) * U * sw, "dweight")
    near(db, wb, (R / 64 + 64) * U * sb, "dbias")


def test_far_rows_of_the_backward(ops):
    """column sums where the only rows that are not zero lie behind the 2^32-th byte: zeros add exactly, so the bound is that of these rows"""
    H, ld = 1001, 40000
    R = 2 ** 31 // ld + 100
    far = torch.zeros(R, ld, device=DEV, dtype=torch.bfloat16)
    last = rnd(50, H, seed=520).to(DEV).bfloat16()
    far[-50:, 7:7 + H] = last
    x, w = far[:, 7:7 + H], rnd(H, seed=521).to(DEV)
    mean, rstd = torch.empty(R, device=DEV), torch.empty(R, device=DEV)
    ops.layer_norm(x, w, mean=mean, rstd=rstd)
    dx, dw, db = ops.layer_norm_bwd(x, x, mean, rstd, w)
    args = [t.cpu() for t in (last, last, mean[-50:], rstd[-50:], w)]
    wx, ww, wb, hat, g = grad64(*args)
    tx, tw, tb = grad_tol(args[0], args[3], hat, g)
    within(dx[-50:], wx, tx * 1.01 + half_step(dx) * wx.abs() * 1.01, "dx")
    within(dw, ww, tw, "dweight")
    within(db, wb, tb, "dbias")
    assert not bool(dx[:-50].any())


def test_layer_norm_and_autograd(ops):
    """by itself the call is outside autograd, as documented; both halves in an autograd.Function give autograd's gradients"""
    R, H = 45, 130
    x, w, b = rnd(R, H, seed=530), 1 + rnd(H, seed=531, scale=0.2), rnd(H, seed=532)
    c = rnd(R, H, seed=533)
    gpu = [t.to(DEV).requires_grad_() for t in (x, w, b)]
    assert not ops.layer_norm(*gpu).requires_grad

    class LayerNorm(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x, weight, bias):
            mean, rstd = (torch.empty(x.shape[0], device=x.device) for _ in range(2))
            ctx.save_for_backward(x, mean, rstd, weight)
            return ops.layer_norm(x, weight, bias, mean=mean, rstd=rstd)

        @staticmethod
        def backward(ctx, dy):
            return ops.layer_norm_bwd(dy.contiguous(), *ctx.saved_tensors)     # a sum's gradient is one value, expanded
    cpu = [t.double().requires_grad_() for t in (x, w, b)]
    for _ in range(2):                                            # gradients of a second pass are added
        y = LayerNorm.apply(*gpu)
        assert y.requires_grad
        (y * c.to(DEV)).sum().backward()
        (norm64(*cpu, 1e-6)[0] * c.double()).sum().backward()
    _, mean, rstd = norm64(x, None, None, 1e-6)
    _, _, _, hat, g = grad64(c, x, mean, rstd, w)
    tols = grad_tol(c, rstd, hat, g)
    # twice the kernel's own bound, the sum of the two passes, and the statistics': mean and rstd are off by 70 u of themselves
    stat = [70 * U * rstd * (g.abs() + hat.abs() * (g * hat).abs().mean(1, keepdim=True) * 3 + g.abs().mean(1, keepdim=True)),
            70 * U * (c.double().abs() * (hat.abs() + rstd * (x.double().abs().mean(1, keepdim=True)))).sum(0), 0]
    for got, want, tol, more in zip(gpu, cpu, tols, stat):
        within(got.grad, want.grad, 2 * (tol + more) + U * want.grad.abs(), "gradient")
    ones = torch.autograd.grad(LayerNorm.apply(*gpu).sum(), gpu[2])[0]
    assert bool((ones == R).all())                                # a sum of ones is exact


@pytest.mark.parametrize("t", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("H", [5, 40, 300, 1000, 3000, 9000, 17000])
def test_layer_norm_in_16_bits_beyond_the_range(ops, t, H):
    """a NaN stays a NaN, what the type's range does not hold becomes an infinity of its sign, as a conversion has it"""
    x = rnd(5, H, seed=540)
    x[1, 3], x[2, 2], x[3, 1] = float("nan"), float("inf"), float("-inf")
    x[0] += 10                                                   # no element close to the mean
    x[0, ::2] -= 20
    big = torch.full((H,), 3e38, device=DEV)
    for src in (x.to(t), x):                                     # 16-bit and fp32 rows
        y = ops.layer_norm(src.to(DEV), big, out_dtype=t).cpu()
        assert y.dtype == t and bool(torch.isnan(y[1:4]).all())
        off = src[0].double() - src[0].double().mean()           # about 10 in magnitude
        assert bool((torch.sign(y[0].double()) == torch.sign(off)).all()) and bool((y[0].double().abs() > 1e37).all())
        if t == torch.float16:
            assert bool(torch.isinf(y[0]).all())
        ok = ops.layer_norm(src.to(DEV), out_dtype=t).cpu()
        assert bool(torch.isfinite(ok[0]).all()) and bool(torch.isfinite(ok[4]).all())
    mean, rstd = torch.zeros(5, device=DEV), torch.full((5,), 1e6, device=DEV)
    mean[0] = float("nan")
    dy = rnd(5, H, seed=541).to(t).to(DEV)
    for k in (1, 500):                                           # few rows in one launch, many in two
        dx = ops.layer_norm_bwd(dy.repeat(k, 1), x.to(t).to(DEV).repeat(k, 1), mean.repeat(k), rstd.repeat(k), big * 1e-30)[0].cpu().view(k, 5, H)
        assert bool(torch.isnan(dx[:, 0]).all()) and bool(torch.isnan(dx[:, 1]).all())
        if t == torch.float16:
            assert not bool((dx[:, 4].abs() == 65504).any()) and bool(torch.isinf(dx[:, 4]).any())


@pytest.mark.parametrize("t", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("M,N,K", [(4, 100, 64), (300, 200, 200), (1600, 1700, 128), (5000, 4200, 128), (5000, 4200, 200)])
def test_gemm_i8_in_16_bits_beyond_the_range(ops, t, M, N, K):
    """every kernel of the product: scales that are not finite, and results that the type's range does not hold"""
    A, W, _, _, _ = operands(M, N, K, seed=550)
    A[:, :K], W[:, :K] = A[:, :K].abs().clamp_min(1), W[:, :K].abs().clamp_min(1)
    sa, sw, b = torch.ones(M), torch.ones(N), torch.zeros(N)
    sa[0], sa[M - 1], sa[M // 2], sa[1] = float("nan"), float("inf"), -1e35, 1e-3
    sw[N // 3] = float("nan")
    b[N - 1] = float("-inf")
    y = ops.gemm_i8(A.to(DEV)[:, :K], sa.to(DEV), W.to(DEV)[:, :K], sw.to(DEV), b.to(DEV), out_dtype=t).cpu()
    nan = torch.zeros(M, N, dtype=torch.bool)
    nan[0], nan[:, N // 3], nan[M - 1, N - 1] = True, True, True
    assert torch.equal(torch.isnan(y), nan)
    assert bool((y[1:M - 1, N - 1] == -math.inf).all()) and bool(((y[M - 1] == math.inf) | nan[M - 1]).all())
    assert bool(torch.isfinite(y[1, :N - 1])[~nan[1, :N - 1]].all())
    if t == torch.float16:
        assert bool(((y[M // 2] == -math.inf) | nan[M // 2]).all()) and not bool((y.abs() == 65504).any())


@pytest.mark.parametrize("t", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("n", [5, 1023, 300000])
def test_adamw_multi_in_16_bits_beyond_the_range(ops, t, bits, n):
    """a norm that is NaN makes every parameter NaN; without clipping a NaN or an infinite parameter stays where it is"""
    for clip in (True, False):
        p = torch.ones(n, device=DEV).to(t)
        p[1], p[n - 1] = float("inf"), torch.finfo(t).max
        g = torch.ones(n, device=DEV)
        g[2] = float("nan")
        g[n - 1] = -1.0
        st = ops.adamw8_state(p) if bits == 8 else (torch.zeros(n, device=DEV), torch.zeros(n, device=DEV))
        args = ops.adamw_multi_args([p], *[[v] for v in st])
        ops.adamw_multi(args, [g], torch.zeros(1, device=DEV, dtype=torch.int32), torch.finfo(t).max / 8 if t == torch.float16 else 1e-3,
                        max_norm=1.0 if clip else None)
        q = p.cpu().float()
        if clip:
            assert bool(torch.isnan(q).all())
            continue
        assert math.isnan(q[2]) and int(torch.isnan(q).sum()) == 1 and math.isinf(q[1])
        if t == torch.float16:                                   # 65504 + 8188
            assert q[n - 1] == math.inf


@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16])
def test_layer_norm_of_very_long_rows(ops, t):
    """rows of 2^26 columns whose mean is far larger than their spread: sums of so many terms keep their digits, as the bounds of
    short rows ask for it; the column sums of very many rows of three columns likewise"""
    H = (1 << 26) + 5
    gen = torch.Generator(DEV).manual_seed(560)
    x = (3.3 + 0.01 * torch.randn(1, H, device=DEV, generator=gen)).to(t)
    mean, rstd = torch.empty(1, device=DEV), torch.empty(1, device=DEV)
    y = ops.layer_norm(x, mean=mean, rstd=rstd)
    want, m, r = norm64(x, None, None, 1e-6)
    size = x.double().abs().mean(1, keepdim=True)
    near(mean.view(1, 1), m, 65 * U * size + U * m.abs(), "mean")
    near(rstd.view(1, 1), r, 70 * U * r + r ** 3 * 65 * U * size ** 2, "rstd")
    near(y, want, norm_tol(x, None, None, m, r) * 1.01 + half_step(y) * want.abs() * 1.01, "y")
    dy = (0.1 + 0.01 * torch.randn(1, H, device=DEV, generator=gen)).to(t)
    dx, _, db = ops.layer_norm_bwd(dy, x, mean, rstd, dbias=torch.empty(H, device=DEV))
    wx, _, _, hat, g = grad64(dy, x, mean, rstd, None)
    near(dx, wx, grad_tol(dy, rstd, hat, g)[0] * 1.01 + half_step(dx) * wx.abs() * 1.01, "dx")
    assert torch.equal(db, dy[0].float())


def test_layer_norm_bwd_of_very_many_short_rows(ops):
    R, H = 3000001, 3
    gen = torch.Generator(DEV).manual_seed(570)
    x, dy = torch.randn(R, H, device=DEV, generator=gen), 0.1 + 1e-4 * torch.randn(R, H, device=DEV, generator=gen)
    mean, rstd = x.double().mean(1).float(), torch.ones(R, device=DEV)
    _, dw, db = ops.layer_norm_bwd(dy, x, mean, rstd, dweight=torch.empty(H, device=DEV), dbias=torch.empty(H, device=DEV))
    _, ww, wb, hat, _ = grad64(dy, x, mean, rstd, None)
    # products of three roundings; a share's sum is rounded once, 64 shares pass at most 2 additions of a slot and 5 of the tree
    near(dw, ww, 11 * U * (dy.double() * hat).abs().sum(0), "dweight")
    near(db, wb, 8 * U * dy.double().abs().sum(0), "dbias")
