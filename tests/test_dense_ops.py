"""linear, segment_matmul and layer_norm against plain float64 arithmetic on the same inputs.

Tolerances are bounds, element by element, with u = half a step of the dtype (relative): a result is rounded once (u |y|); a float32
sum of n products is off by at most n steps of 2^-23 of the sum of their absolute values (a matrix instruction may truncate where it
adds: a whole step); a float32 product of split operands is six such products plus at most 2^-23 of |ab| left out.  The gradient of an
activation is taken at z rounded to the dtype: |act''| <= 0.8 (gelu) or 0.5 (silu) times that rounding; relu's may be 0 or 1 where |z| is
below the sum's own error.  gelu and its slope are polynomials: for 16-bit results 2^-15 of the value and 2^-15 absolute (what their fits
leave), for float32 below 2^-20 like the other activations.
"""
import math

import pytest
import torch

import geot_amd as geot

gpu = pytest.mark.gpu
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
IDS = ["f32", "f16", "bf16"]
STEP = 2.0 ** -23
CURVATURE = {"none": 0.0, "relu": 0.0, "gelu": 0.8, "silu": 0.5}


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def terms(n, dtype):
    return (6 * n + 16 if dtype == torch.float32 else n + 16) * STEP


def rand(*shape, dtype, seed, scale=1.0, device="cuda"):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(dtype).to(device)


def act64(z, name):
    if name == "relu":
        return z.clamp(min=0), (z > 0).double()
    if name == "gelu":
        cdf = torch.special.ndtr(z)
        return z * cdf, cdf + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if name == "silu":
        s = torch.sigmoid(z)
        return z * s, s * (1 + z * (1 - s))
    return z, torch.ones_like(z)


def close(got, want, tol, what):
    assert got.shape == want.shape, (what, got.shape, want.shape)
    err = (got.double() - want).abs()
    bad = ~(err <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((err / tol.clamp(min=1e-300)).max()):.3g} x the bound"


class LinearReference:
    """y and, given dy, the gradients in float64 with the bound of each."""

    def __init__(self, x, w, b, r, act, dy=None):
        dt, u = x.dtype, half_step(x.dtype)
        tiny = torch.finfo(dt).tiny
        x, w = x.double().reshape(-1, x.shape[-1]), w.double()
        m, k, n = x.shape[0], x.shape[1], w.shape[0]
        z = x @ w.t().contiguous()
        size = x.abs() @ w.abs().t().contiguous()
        if b is not None:
            z, size = z + b.double(), size + b.double().abs()
        e_z = terms(k, dt) * size
        f, slope = act64(z, act)
        fit = 2.0 ** -15 if act == "gelu" and dt != torch.float32 else 0.0
        self.y, self.e_y = f, 1.2 * e_z + (2.0 ** -20 + fit) * f.abs()
        if r is not None:
            r = r.double().reshape(m, n)
            self.y, self.e_y = f + r, self.e_y + STEP * (f.abs() + r.abs())
        self.e_y = self.e_y + u * (self.y.abs() + self.e_y) + tiny
        if dy is None:
            return
        dy = dy.double().reshape(m, n)
        dz = dy * slope
        e_dz = torch.zeros_like(dz)
        if act != "none":
            e_slope = CURVATURE[act] * (e_z + u * z.abs() + tiny) + 2.0 ** -20 * (slope.abs() + z.abs() / 2) + fit
            if act == "relu":
                e_slope = (z.abs() <= e_z + tiny).double()
            e_dz = dy.abs() * e_slope + u * dz.abs() + tiny
        hi = dz.abs() + e_dz

        def bound(e, s, n_terms, v):
            e = e + terms(n_terms, dt) * s
            return e + u * (v.abs() + e) + tiny

        self.dx = dz @ w
        self.e_dx = bound(e_dz @ w.abs(), hi @ w.abs(), n, self.dx)
        self.dw = dz.t().contiguous() @ x
        self.e_dw = bound(e_dz.t().contiguous() @ x.abs(), hi.t().contiguous() @ x.abs(), m, self.dw)
        self.db = dz.sum(0)
        self.e_db = bound(e_dz.sum(0), hi.sum(0), m, self.db)


LINEAR_SHAPES = [(1, 1, 1), (5, 16, 32), (1, 520, 96), (3, 64, 1000), (128, 128, 128), (129, 65, 33), (300, 602, 256), (257, 64, 130), (64, 200, 72),
                 (200, 7, 128), (1000, 33, 64), (31, 1024, 40), (2, 120, 1990), (70, 4100, 48), (700, 24, 80)]


# ---- refusals: no GPU needed ------------------------------------------------------------------------------------------------------
def test_refusals():
    x, w = torch.zeros(4, 6), torch.zeros(5, 6)
    with pytest.raises(RuntimeError, match="CPU tensors are not supported"):
        geot.linear(x, w)
    with pytest.raises(RuntimeError, match="CPU tensors are not supported"):
        geot.linear(x.requires_grad_(), w)
    x = torch.zeros(4, 6)
    with pytest.raises(RuntimeError, match="6 features a row, weight takes 7"):
        geot.linear(x, torch.zeros(5, 7))
    with pytest.raises(RuntimeError, match="at least 1 dimensional"):
        geot.linear(torch.zeros(()), w)
    with pytest.raises(RuntimeError, match="2 dimensional"):
        geot.linear(x, torch.zeros(5, 6, 1))
    with pytest.raises(RuntimeError, match="expected weight of dtype Float but found Half"):
        geot.linear(x, w.half())
    with pytest.raises(RuntimeError, match="bias must have one value per output feature"):
        geot.linear(x, w, torch.zeros(6))
    with pytest.raises(RuntimeError, match="residual must have the output's shape"):
        geot.linear(x, w, residual=torch.zeros(1, 5))
    with pytest.raises(RuntimeError, match="activation argument must be either none, relu, gelu or silu, got tanh"):
        geot.linear(x, w, activation="tanh")

    w3, ptr = torch.zeros(3, 6, 5), torch.tensor([0, 1, 2, 4])
    with pytest.raises(RuntimeError, match="CPU tensors are not supported"):
        geot.segment_matmul(x, ptr, w3)
    with pytest.raises(RuntimeError, match="groups \\+ 1 = 4 row offsets"):
        geot.segment_matmul(x, ptr[:-1], w3)
    with pytest.raises(RuntimeError, match="expected scalar type Long but found Int"):
        geot.segment_matmul(x, ptr.int(), w3)
    with pytest.raises(RuntimeError, match="x must be 2 dimensional"):
        geot.segment_matmul(x[None], ptr, w3)
    with pytest.raises(RuntimeError, match="weight takes 7"):
        geot.segment_matmul(x, ptr, torch.zeros(3, 7, 5))
    with pytest.raises(RuntimeError, match="bias must be"):
        geot.segment_matmul(x, ptr, w3, torch.zeros(5))

    with pytest.raises(RuntimeError, match="CPU tensors are not supported"):
        geot.layer_norm(x)
    with pytest.raises(RuntimeError, match="one value per feature"):
        geot.layer_norm(x, torch.ones(5))
    with pytest.raises(RuntimeError, match="one dtype"):
        geot.layer_norm(x.half(), torch.ones(6), torch.ones(6).half())
    with pytest.raises(RuntimeError, match="expected weight and bias of dtype Half or Float but found Double"):
        geot.layer_norm(x.half(), torch.ones(6).double())


def test_refused_abi_calls():
    """What the C ABI refuses before it touches anything."""
    L = geot._lib.load()
    einval, eworkspace, eunsupported = -1, -2, -4
    assert L.geot_linear(None, 4, None, None, None, 0, None, None, -1, 4, 4, 0, 0, None, 0, None) == einval
    assert L.geot_linear(None, 4, None, None, None, 0, None, None, 2, 4, 4, 0, 0, None, 0, None) == einval
    assert L.geot_linear(None, 4, None, None, None, 0, None, None, 0, 4, 4, 9, 0, None, 0, None) == einval
    assert L.geot_linear(16, 4, 16, None, None, 0, None, 16, 2, 4, 4, 0, 1, None, 0, None) == eunsupported       # (float64: refused before any launch)
    assert L.geot_segment_matmul(16, 4, 16, 16, None, 16, 2, 65536, 4, 4, 0, None, 0, None) == einval
    need = L.geot_segment_matmul_workspace_bytes(17, 2, 4096, 128, 0)
    assert need > 0 and L.geot_segment_matmul_workspace_bytes(1_000_000, 2, 4096, 128, 0) == 0
    assert L.geot_segment_matmul(16, 4096, 16, 16, None, 16, 17, 2, 4096, 128, 0, 16, need - 4, None) == eworkspace
    need = L.geot_linear_grad_weight_workspace_bytes(1_000_000, 64, 64, 0)
    assert need > 0 and L.geot_linear_grad_weight_workspace_bytes(100, 64, 64, 0) == 0
    assert L.geot_linear_grad_weight(16, 16, 64, 16, 16, 1_000_000, 64, 64, 0, 16, need - 4, None) == eworkspace
    assert L.geot_layer_norm(16, 4, None, None, 16, None, 2, 4, 1e-5, 1, 1, None) == eunsupported
    assert L.geot_layer_norm_backward(16, 4, None, 16, 16, 16, 16, 16, 2, 4, 0, 0, 16, 4, None) == eworkspace
    assert L.geot_layer_norm_backward(16, 4, None, 16, 16, 16, 16, None, 2, 4, 0, 0, 16, 1 << 20, None) == einval


def test_fake_shapes():
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        x = torch.empty(3, 4, 8, dtype=torch.bfloat16, device="cuda")
        w = torch.empty(6, 8, dtype=torch.bfloat16, device="cuda")
        assert geot.linear(x, w, activation="gelu").shape == (3, 4, 6)
        # a narrow layer's pre-activation is computed again, a wide one's is kept (unless y has its sign)
        assert torch.ops.geot_dense.linear_train(x, w, None, None, "gelu")[1].numel() == 0
        xw, ww = torch.empty(3, 4, 300, dtype=torch.bfloat16, device="cuda"), torch.empty(6, 300, dtype=torch.bfloat16, device="cuda")
        y, z = torch.ops.geot_dense.linear_train(xw, ww, None, None, "gelu")
        assert z.shape == y.shape and torch.ops.geot_dense.linear_train(xw, ww, None, None, "relu")[1].numel() == 0
        assert geot.layer_norm(x, w[0].float()).shape == x.shape
        assert torch.ops.geot_dense.layer_norm_train(x, w[0].float(), None, 1e-5)[1].shape == (3, 12)
        assert geot.segment_matmul(x[0], torch.empty(3, dtype=torch.int64, device="cuda"), torch.empty(2, 8, 5, dtype=torch.bfloat16, device="cuda")).shape == (4, 5)


# ---- linear -----------------------------------------------------------------------------------------------------------------------
@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("m,k,n", LINEAR_SHAPES)
def test_linear(m, k, n, dtype):
    for i, (act, bias, res) in enumerate([("none", False, False), ("relu", True, True), ("relu", True, False), ("gelu", True, True), ("silu", False, True)]):
        seed = 10 * (m + 3 * k + 7 * n) + i
        x, w = rand(m, k, dtype=dtype, seed=seed), rand(n, k, dtype=dtype, seed=seed + 1, scale=k ** -0.5)
        b = rand(n, dtype=dtype, seed=seed + 2) if bias else None
        r = rand(m, n, dtype=dtype, seed=seed + 3) if res else None
        dy = rand(m, n, dtype=dtype, seed=seed + 4)
        ref = LinearReference(x, w, b, r, act, dy)
        y = geot.linear(x, w, b, residual=r, activation=act)
        close(y, ref.y, ref.e_y, f"y {act}")
        leaves = [t.requires_grad_() for t in (x, w, b, r) if t is not None]
        yt = geot.linear(x, w, b, residual=r, activation=act)
        assert torch.equal(yt, y)
        grads = list(torch.autograd.grad(yt, leaves, dy))
        close(grads[0], ref.dx, ref.e_dx, f"dx {act}")
        close(grads[1], ref.dw, ref.e_dw, f"dw {act}")
        if bias:
            close(grads[2], ref.db, ref.e_db, f"db {act}")
        if res:
            assert torch.equal(grads[-1], dy)


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_linear_many_rows(dtype):
    """Rows split over workgroups and joined in the weight's gradient; also twice, bit for bit."""
    m, k, n = 70_001, 40, 24
    x, w, b, dy = (rand(*s, dtype=dtype, seed=i) for i, s in enumerate([(m, k), (n, k), (n,), (m, n)]))
    ref = LinearReference(x, w, b, None, "silu", dy)
    leaves = [t.requires_grad_() for t in (x, w, b)]
    runs = []
    for _ in range(2):
        y = geot.linear(x, w, b, activation="silu")
        runs.append([y.detach(), *torch.autograd.grad(y, leaves, dy)])
    for a, c in zip(*runs):
        assert torch.equal(a, c)
    for got, want, tol, what in zip(runs[0], (ref.y, ref.dx, ref.dw, ref.db), (ref.e_y, ref.e_dx, ref.e_dw, ref.e_db), ("y", "dx", "dw", "db")):
        close(got, want, tol, what)


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_linear_partial_gradients(dtype):
    """Only what is asked for: x alone, the weight alone, the bias alone, the residual alone."""
    m, k, n = 70, 20, 36
    x, w, b, r, dy = (rand(*s, dtype=dtype, seed=i) for i, s in enumerate([(m, k), (n, k), (n,), (m, n), (m, n)]))
    ref = LinearReference(x, w, b, r, "gelu", dy)
    for which, want, tol in ((0, ref.dx, ref.e_dx), (1, ref.dw, ref.e_dw), (2, ref.db, ref.e_db), (3, dy.double(), torch.zeros_like(ref.y))):
        args = [t.detach().clone() for t in (x, w, b, r)]
        args[which].requires_grad_()
        y = geot.linear(args[0], args[1], args[2], residual=args[3], activation="gelu")
        (g,) = torch.autograd.grad(y, [args[which]], dy)
        close(g, want, tol, f"leaf {which}")


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_linear_empty_sizes(dtype):
    for m, k, n in ((0, 8, 8), (7, 0, 5), (7, 8, 0), (0, 0, 0)):
        x, w, b, r = (torch.ones(*s, dtype=dtype, device="cuda", requires_grad=True) for s in ((m, k), (n, k), (n,), (m, n)))
        y = geot.linear(x, w, b, residual=r, activation="relu")
        assert y.shape == (m, n) and bool((y == 2).all())
        dx, dw, db = torch.autograd.grad(y, [x, w, b], torch.ones_like(y))
        assert dx.shape == x.shape and dw.shape == w.shape and db.shape == b.shape
        assert bool((dx == n).all()) and bool((dw == (m if k else 0)).all()) and bool((db == m).all())


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_linear_layouts(dtype):
    """Views: rows of a wider table, an odd offset, transposed operands, more dimensions, expanded residual and gradient."""
    m, k, n = 150, 37, 45
    table = rand(m, 96, dtype=dtype, seed=1)
    flat = rand(m * k + 3, dtype=dtype, seed=2)
    w = rand(n, k, dtype=dtype, seed=3, scale=0.2)
    b = rand(n, dtype=dtype, seed=4)
    wide_r = rand(m, 2 * n, dtype=dtype, seed=5)
    for x in (table[:, 5:5 + k], table[:, ::2][:, :k], flat[3:].view(m, k), rand(k, m, dtype=dtype, seed=6).t()):
        for r in (None, wide_r[:, n:], wide_r[0, :n].expand(m, n), rand(n, m, dtype=dtype, seed=7).t()):
            ref = LinearReference(x, w, b, r, "gelu")
            close(geot.linear(x, w, b, residual=r, activation="gelu"), ref.y, ref.e_y, "y")
    x = table[:, 5:5 + k]
    for weight in (rand(k, n, dtype=dtype, seed=8, scale=0.2).t(), rand(2 * n, k, dtype=dtype, seed=9, scale=0.2)[::2]):
        ref = LinearReference(x, weight, b, None, "none")
        close(geot.linear(x, weight, b), ref.y, ref.e_y, "y, strided weight")
    x3 = rand(5, 6, 30, dtype=dtype, seed=10).transpose(0, 1).requires_grad_()
    w3 = rand(n, 30, dtype=dtype, seed=11, scale=0.2).requires_grad_()
    y = geot.linear(x3, w3, activation="silu")
    assert y.shape == (6, 5, n)
    dy = rand(n, dtype=dtype, seed=12).expand(6, 5, n)
    ref = LinearReference(x3, w3, None, None, "silu", dy)
    dx, dw = torch.autograd.grad(y, [x3, w3], dy)
    close(y.reshape(30, n), ref.y, ref.e_y, "y, three dimensions")
    close(dx.reshape(30, 30), ref.dx, ref.e_dx, "dx, expanded gradient")
    close(dw, ref.dw, ref.e_dw, "dw, expanded gradient")
    x1 = rand(30, dtype=dtype, seed=13)
    ref = LinearReference(x1, w3, None, None, "none")
    close(geot.linear(x1, w3.detach()).view(1, n), ref.y, ref.e_y, "one row without a row dimension")


@gpu
def test_linear_float32_keeps_24_bits():
    """A weight with one entry a row selects and scales: the product of two 24-bit significands may be off by one last place of float32
    (half a step of rounding, 2^-23 left out of the split product), and by nothing where the factor is a power of two."""
    m, k = 200, 96
    x = rand(m, k, dtype=torch.float32, seed=0) * torch.logspace(-20, 20, k, device="cuda")
    perm = torch.randperm(k, generator=torch.Generator().manual_seed(1)).cuda()
    for w, exact in ((torch.full((k,), -0.125, device="cuda"), True), (rand(k, dtype=torch.float32, seed=2), False)):
        weight = torch.zeros(k, k, device="cuda")
        weight[torch.arange(k, device="cuda"), perm] = w
        got, want = geot.linear(x, weight).double(), x[:, perm].double() * w.double()
        if exact:
            assert torch.equal(got, want)
        assert bool(((got - want).abs() <= 2.0 ** -22 * want.abs()).all())
    # a factor below 2^-110: its parts below the smallest bfloat16, 2^-133, are lost
    for e in (-140, -127, -115, -100):
        small = x / x.abs().clamp(min=1e-30) * 2.0 ** e * torch.linspace(1, 2, k, device="cuda")
        err = (geot.linear(small, torch.eye(k, device="cuda") * 2.0 ** 30).double() - small.double() * 2.0 ** 30).abs()
        assert bool((err <= 2.0 ** (30 - 133) + 2.0 ** -22 * 2.0 ** 30 * small.double().abs()).all())


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_linear_infinities_and_nan(dtype):
    """They come out as in ordinary arithmetic, and in their own rows and columns only."""
    m, k, n = 140, 70, 90
    x, w = rand(m, k, dtype=dtype, seed=0), rand(n, k, dtype=dtype, seed=1)
    clean = geot.linear(x, w)
    inf, big = float("inf"), torch.finfo(dtype).max
    x2, w2 = x.clone(), w.clone()
    x2[3, 5], x2[130, 0], x2[131, 69], x2[7, 7], w2[80, 3] = inf, -inf, float("nan"), big, inf
    w2[2, 5] = 0                                     # inf * 0
    want = (x2.double() @ w2.double().t().contiguous())
    got = geot.linear(x2, w2)
    rows = torch.ones(m, dtype=torch.bool, device="cuda")
    rows[[3, 7, 130, 131]] = False
    cols = torch.ones(n, dtype=torch.bool, device="cuda")
    cols[[2, 80]] = False
    assert torch.equal(got[rows][:, cols], clean[rows][:, cols])
    sure = ~torch.isfinite(want)
    assert torch.equal(torch.isnan(got)[sure], torch.isnan(want)[sure])
    inf_places = torch.isinf(want)
    assert torch.equal(got.double()[inf_places], want[inf_places])
    small = want.abs() < big / 4                     # (products that fit again, e.g. big * 1e-3)
    rounded = torch.isfinite(want) & small
    size = x2.double().abs() @ w2.double().abs().t().contiguous()
    tol = terms(k, dtype) * size + half_step(dtype) * want.abs() + 1e-7
    assert bool(((got.double() - want).abs() <= tol)[rounded].all())
    # the gradient of the weight: rows 3, 130, 131 reach every output's columns 5, 0, 69
    xg, wg = x2.clone(), w.clone().requires_grad_()
    dy = rand(m, n, dtype=dtype, seed=2)
    (dw,) = torch.autograd.grad(geot.linear(xg, wg), [wg], dy)
    want = dy.double().t().contiguous() @ x2.double()
    assert torch.equal(torch.isnan(dw), torch.isnan(want)) and torch.equal(dw.double()[:, [0, 5]], want[:, [0, 5]])


@gpu
def test_linear_past_32_bits():
    """Row offsets beyond 2^31 elements."""
    m, k, n = 2_200_000, 1000, 8
    x = torch.zeros(m, k, dtype=torch.bfloat16, device="cuda")
    tail = rand(200, k, dtype=torch.bfloat16, seed=1)
    x[-200:] = tail
    w = rand(n, k, dtype=torch.bfloat16, seed=2, scale=0.03)
    ref = LinearReference(tail, w, None, None, "none")
    close(geot.linear(x, w)[-200:], ref.y, ref.e_y, "last rows")
    dy = torch.zeros(m, n, dtype=torch.bfloat16, device="cuda")
    dy[-200:] = rand(200, n, dtype=torch.bfloat16, seed=3)
    ref = LinearReference(tail, w, None, None, "none", dy[-200:])
    w.requires_grad_()
    (dw,) = torch.autograd.grad(geot.linear(x, w), [w], dy)
    close(dw, ref.dw, ref.e_dw, "dw")


# ---- segment_matmul -----------------------------------------------------------------------------------------------------------------
def segment_reference(x, ptr, w, b, dy):
    """Group by group, as linear with the group's transposed matrix."""
    m, groups, n = x.shape[0], w.shape[0], w.shape[2]
    z64 = lambda *s: torch.zeros(*s, dtype=torch.float64, device=x.device)  # noqa: E731
    out = {k: (z64(*s), z64(*s)) for k, s in (("y", (m, n)), ("dx", x.shape), ("dw", w.shape), ("db", (groups, n)))}
    for g in range(groups):
        lo, hi = ptr[g], ptr[g + 1]
        if lo == hi:
            continue
        ref = LinearReference(x[lo:hi], w[g].t(), None if b is None else b[g], None, "none", dy[lo:hi])
        for key, v, e, at in (("y", ref.y, ref.e_y, slice(lo, hi)), ("dx", ref.dx, ref.e_dx, slice(lo, hi)), ("dw", ref.dw.t(), ref.e_dw.t(), g),
                              ("db", ref.db, ref.e_db, g)):
            out[key][0][at], out[key][1][at] = v, e
    return out


SEGMENTS = [
    ([0, 5], 16, 8),                                        # one group
    ([0, 0, 3, 3, 3, 130, 131, 131], 20, 33),               # empty groups in front, between and behind
    ([0, 128, 256, 257, 600], 64, 128),                     # whole tiles
    ([7, 60, 60, 190], 37, 70),                             # rows in front of the first group
    ([0, 90, 101], 130, 65),                                # rows behind the last group (101 of 150)
    ([0, 0, 0], 8, 8),                                      # no group has rows
    (list(range(0, 301, 3)), 24, 40),                       # 100 groups of 3 rows
    ([0, 1, 2, 3, 4], 512, 96),                             # one row a group
    ([0, 3000, 3001, 9000], 72, 48),                        # groups of several chunks beside tiny ones
    ([2, 19, 19, 20], 1500, 700),                           # few rows, long reductions both ways: split over workgroups (25 rows)
]


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("case", range(len(SEGMENTS)))
def test_segment_matmul(case, dtype):
    rows, k, n = SEGMENTS[case]
    groups, m = len(rows) - 1, {4: 150, 5: 40, 9: 25}.get(case, rows[-1])
    x, w, b, dy = (rand(*s, dtype=dtype, seed=100 * case + i, scale=sc) for i, (s, sc) in enumerate(
        [((m, k), 1), ((groups, k, n), k ** -0.5), ((groups, n), 1), ((m, n), 1)]))
    ptr = torch.tensor(rows, device="cuda")
    for bias in (None, b):
        ref = segment_reference(x.detach(), rows, w.detach(), None if bias is None else b.detach(), dy)
        with torch.no_grad():
            close(geot.segment_matmul(x, ptr, w, bias), *ref["y"], "y")
        leaves = [t.requires_grad_() for t in (x, w) + (() if bias is None else (b,))]
        y = geot.segment_matmul(x, ptr, w, bias)
        grads = torch.autograd.grad(y, leaves, dy)
        again = torch.autograd.grad(geot.segment_matmul(x, ptr, w, bias), leaves, dy)
        close(y, *ref["y"], "y")
        for key, g, g2 in zip(("dx", "dw", "db"), grads, again):
            close(g, *ref[key], key)
            assert torch.equal(g, g2)
    # the bias's gradient alone
    (db,) = torch.autograd.grad(geot.segment_matmul(x.detach(), ptr, w.detach(), b), [b], dy)
    close(db, *ref["db"], "db alone")


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_segment_matmul_groups_keep_apart(dtype):
    """NaN rows of one group reach no other; a strided x; a pointer array that is itself a view."""
    rows, k, n = [0, 40, 41, 200, 200, 333], 36, 50
    table = rand(333, 80, dtype=dtype, seed=1)
    x = table[:, 4:4 + k]
    w, dy = rand(5, k, n, dtype=dtype, seed=2, scale=0.2), rand(333, n, dtype=dtype, seed=3)
    ptr = torch.stack([torch.tensor(rows), torch.zeros(6, dtype=torch.int64)], 1).cuda()[:, 0]
    ref = segment_reference(x, rows, w, None, dy)
    bad = x.clone()
    bad[41:200] = float("nan")
    w.requires_grad_()
    y = geot.segment_matmul(bad, ptr, w)
    (dw,) = torch.autograd.grad(y, [w], dy)
    keep = torch.ones(333, dtype=torch.bool, device="cuda")
    keep[41:200] = False
    close(y[keep], ref["y"][0][keep], ref["y"][1][keep], "y of the other groups")
    assert bool(torch.isnan(y[~keep]).all())
    others = [0, 1, 3, 4]
    close(dw[others], ref["dw"][0][others], ref["dw"][1][others], "dw of the other groups")
    close(geot.segment_matmul(x, ptr, w.detach()), *ref["y"], "y, strided x")


@gpu
def test_segment_matmul_bad_pointers_stay_inside():
    """Entries out of range are clamped: as if they were 0 or the row count.  (Bounds: every row the kernels touch is in [0, rows).)"""
    m, k, n = 100, 16, 24
    x, w = rand(m, k, dtype=torch.float32, seed=1), rand(2, k, n, dtype=torch.float32, seed=2)
    got = geot.segment_matmul(x, torch.tensor([-5, 60, 10 ** 12], device="cuda"), w)
    assert torch.equal(got, geot.segment_matmul(x, torch.tensor([0, 60, m], device="cuda"), w))


@gpu
def test_segment_matmul_no_groups():
    x, w = torch.ones(9, 4, device="cuda", requires_grad=True), torch.ones(0, 4, 6, device="cuda", requires_grad=True)
    y = geot.segment_matmul(x, torch.tensor([3], device="cuda"), w)
    assert y.shape == (9, 6) and bool((y == 0).all())
    dx, dw = torch.autograd.grad(y, [x, w], torch.ones_like(y))
    assert bool((dx == 0).all()) and dw.shape == (0, 4, 6)
    empty = geot.segment_matmul(torch.ones(0, 4, device="cuda"), torch.tensor([0, 0], device="cuda"), torch.ones(1, 4, 6, device="cuda"))
    assert empty.shape == (0, 6)


# ---- layer_norm -----------------------------------------------------------------------------------------------------------------------
NORM_SHAPES = [(1, 1), (3, 5), (1000, 16), (70, 64), (33, 65), (257, 128), (40, 200), (65, 256), (30, 300), (9, 512), (17, 602), (6, 1024), (5, 1025),
               (12, 2048), (3, 2049), (7, 4096), (2, 5000), (3, 8192), (2, 8193), (70, 10_007)]


def norm_reference(x, w, b, dy, eps=1e-5):
    u, d = half_step(x.dtype), x.shape[-1]
    n = (64 + d / 256) * 2.0 ** -24                          # longest chain of float32 additions of a row's sum
    x, dy = x.double().reshape(-1, d), dy.double().reshape(-1, d)
    w64 = torch.ones(d, dtype=torch.float64, device=x.device) if w is None else w.double()
    b64 = torch.zeros_like(w64) if b is None else b.double()
    var, mean = torch.var_mean(x, -1, unbiased=False, keepdim=True)
    s = (var + eps).rsqrt()
    h = (x - mean) * s
    e_h = n * (h.abs() + 1)
    y, g = h * w64 + b64, dy * w64
    q, m = (g * h).mean(-1, keepdim=True), g.mean(-1, keepdim=True)
    dx = s * (g - m - h * q)
    size = g.abs() + g.abs().mean(-1, keepdim=True) + h.abs() * (g * h).abs().mean(-1, keepdim=True)
    e_dx = s * (3 * n * size + e_h * q.abs() + h.abs() * (g.abs() * e_h).mean(-1, keepdim=True))
    rows = x.shape[0] * 2.0 ** -24
    dw, db = (dy * h).sum(0), dy.sum(0)
    pu = u if w is None and b is None else half_step((w if w is not None else b).dtype)

    def fin(e, v, uu):
        return e + uu * (v.abs() + e) + 1e-30 + (torch.finfo(torch.float16).tiny if uu == 2.0 ** -11 else 0)

    return {"y": (y, fin(e_h * w64.abs() + 2 * STEP * y.abs(), y, u)), "dx": (dx, fin(e_dx, dx, u)),
            "dw": (dw, fin((rows + n) * (dy * h).abs().sum(0) + (dy.abs() * e_h).sum(0), dw, pu)), "db": (db, fin((rows + n) * dy.abs().sum(0), db, pu))}


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("m,d", NORM_SHAPES)
def test_layer_norm(m, d, dtype):
    x, dy = rand(m, d, dtype=dtype, seed=m + d, scale=1.5), rand(m, d, dtype=dtype, seed=m + d + 1)
    for pdtype in {dtype, torch.float32}:
        w, b = rand(d, dtype=pdtype, seed=2), rand(d, dtype=pdtype, seed=3)
        for weight, bias in ((w, b), (None, None), (w, None), (None, b)):
            ref = norm_reference(x.detach(), None if weight is None else w.detach(), None if bias is None else b.detach(), dy)
            with torch.no_grad():
                close(geot.layer_norm(x, weight, bias), *ref["y"], "y")
            leaves = [t.requires_grad_() for t in (x, weight, bias) if t is not None]
            y = geot.layer_norm(x, weight, bias)
            close(y, *ref["y"], "y")
            names = ["dx"] + ["dw"] * (weight is not None) + ["db"] * (bias is not None)
            grads = torch.autograd.grad(y, leaves, dy)
            again = torch.autograd.grad(geot.layer_norm(x, weight, bias), leaves, dy)
            for key, g, g2 in zip(names, grads, again):
                close(g, *ref[key], key)
                assert torch.equal(g, g2)
            x = x.detach()


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_layer_norm_many_rows(dtype):
    m, d = 60_011, 24
    x, dy, w, b = (rand(*s, dtype=dtype, seed=i) for i, s in enumerate([(m, d), (m, d), (d,), (d,)]))
    ref = norm_reference(x, w, b, dy)
    y = geot.layer_norm(x.requires_grad_(), w.requires_grad_(), b.requires_grad_())
    close(y, *ref["y"], "y")
    for key, g in zip(("dx", "dw", "db"), torch.autograd.grad(y, [x, w, b], dy)):
        close(g, *ref[key], key)


@gpu
@pytest.mark.parametrize("d", [48, 700, 3000, 9000])
def test_layer_norm_far_from_zero(d):
    """Rows with mean 1e4 and spread 1: the same bound as rows around zero."""
    x = rand(20, d, dtype=torch.float32, seed=1) + 1e4
    dy = rand(20, d, dtype=torch.float32, seed=2)
    ref = norm_reference(x, None, None, dy)
    x.requires_grad_()
    y = geot.layer_norm(x)
    close(y, *ref["y"], "y")
    close(torch.autograd.grad(y, [x], dy)[0], *ref["dx"], "dx")


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_layer_norm_edges(dtype):
    """Constant rows, rows with NaN or an infinity, empty sizes, strided and offset rows, more dimensions."""
    x = rand(50, 96, dtype=dtype, seed=1)
    x[3], x[10, 4], x[11, 5] = 2.5, float("nan"), float("inf")
    y = geot.layer_norm(x)
    # a constant row: x - m is at most one rounding of the mean (2^-23 * 2.5), taken off again up to 2^-24 of itself, times 1 / sqrt(eps) = 317
    assert bool((y[3].abs() <= 2.0 ** -23 * 2.5 * 2.0 ** -24 * 317).all())
    assert bool(torch.isnan(y[10]).all()) and bool(torch.isnan(y[11]).all())
    keep = [i for i in range(50) if i not in (3, 10, 11)]
    ref = norm_reference(x[keep], None, None, x[keep])
    close(y[keep], *ref["y"], "other rows")
    for m, d in ((0, 5), (4, 0)):
        t = [torch.ones(*s, dtype=dtype, device="cuda", requires_grad=True) for s in ((m, d), (d,), (d,))]
        y = geot.layer_norm(*t)
        g = torch.autograd.grad(y, t, torch.ones_like(y))
        assert y.shape == (m, d) and [a.shape for a in g] == [a.shape for a in t] and all(bool((a == 0).all()) for a in g)
    table = rand(40, 150, dtype=dtype, seed=2)
    for v in (table[:, 7:107], table[::2, 1:], rand(30, 40, dtype=dtype, seed=3).t(), rand(4, 5, 33, dtype=dtype, seed=4).transpose(0, 1)):
        v = v.detach().requires_grad_()
        dy = rand(v.shape[-1], dtype=dtype, seed=5).expand(v.shape)
        ref = norm_reference(v.detach(), None, None, dy)
        y = geot.layer_norm(v)
        close(y.reshape(-1, v.shape[-1]), *ref["y"], "y")
        close(torch.autograd.grad(y, [v], dy)[0].reshape(-1, v.shape[-1]), *ref["dx"], "dx")
    with pytest.raises(RuntimeError, match="not implemented for 'Double'"):
        geot.layer_norm(x.double())
    with pytest.raises(RuntimeError, match="not implemented for 'Double'"):
        geot.linear(x.double(), x.double())


# ---- together, and as programs call them ----------------------------------------------------------------------------------------------
def _typed_layer(x, edges, ptr, wrel, wself, bself, gamma, beta, n):
    """One layer of a heterogeneous graph: messages through their relation's matrix, summed per destination, a self transform with the
    activation and a skip connection, the normalisation."""
    src, dst, order = edges
    msg = geot.segment_matmul(x.index_select(0, src), ptr, wrel)
    agg = geot.index_scatter(0, msg.index_select(0, order), dst, "sum", True)
    agg = torch.nn.functional.pad(agg, (0, 0, 0, n - agg.shape[0]))
    h = geot.linear(x, wself, bself, residual=agg, activation="silu")
    return geot.layer_norm(h, gamma, beta)


def _typed_layer64(x, edges, rows, wrel, wself, bself, gamma, beta, n):
    src, dst, order = edges
    g = x.index_select(0, src)
    msg = torch.cat([g[a:b] @ wrel[i] for i, (a, b) in enumerate(zip(rows[:-1], rows[1:]))])
    agg = torch.zeros(n, msg.shape[1], dtype=x.dtype, device=x.device).index_add(0, dst, msg.index_select(0, order))
    z = x @ wself.t() + bself
    h = z * torch.sigmoid(z) + agg
    mu = h.mean(-1, keepdim=True)
    return (h - mu) / ((h - mu).square().mean(-1, keepdim=True) + 1e-5).sqrt() * gamma + beta


def _typed_problem(seed=0, n=400, e=3000, f=48):
    g = torch.Generator().manual_seed(seed)
    rel, dst = torch.sort(torch.randint(0, 5, (e,), generator=g)).values, torch.randint(0, n, (e,), generator=g)
    rows = [0] + torch.cumsum(torch.bincount(rel, minlength=6), 0).tolist()          # (relation 5 has no edges)
    order = torch.argsort(dst, stable=True)
    edges = [t.cuda() for t in (torch.randint(0, n, (e,), generator=g), dst[order], order)]
    tensors = [rand(*s, dtype=torch.float32, seed=seed + i, scale=sc) for i, (s, sc) in enumerate(
        [((n, f), 1), ((6, f, f), 0.1), ((f, f), 0.14), ((f,), 0.3), ((f,), 1), ((f,), 1)])]
    return n, edges, rows, torch.tensor(rows, device="cuda"), tensors


@gpu
def test_a_layer_of_all_of_them():
    """Forward and every gradient of the layer against float64 autograd.  float32 throughout: sums of at most 3000 terms, results of size 1
    (normalised rows): 2e-4 is over 10 x their first-order bound at the conditioning of these inputs (row spreads 0.5 to 3)."""
    n, edges, rows, ptr, tensors = _typed_problem()
    leaves = [t.requires_grad_() for t in tensors]
    y = _typed_layer(tensors[0], edges, ptr, *tensors[1:], n)
    dy = rand(*y.shape, dtype=torch.float32, seed=99)
    grads = torch.autograd.grad(y, leaves, dy)
    leaves64 = [t.detach().double().requires_grad_() for t in tensors]
    y64 = _typed_layer64(leaves64[0], edges, rows, *leaves64[1:], n)
    grads64 = torch.autograd.grad(y64, leaves64, dy.double())
    assert float((y.double() - y64).abs().max()) <= 2e-4
    for g, g64 in zip(grads, grads64):
        assert float((g.double() - g64).abs().max()) <= 2e-4 * float(g64.abs().max())


@gpu
@pytest.mark.parametrize("op", ["linear", "segment_matmul", "layer_norm"])
def test_gradients_against_differences(op):
    """<gradient, v> against (f(+h v) - f(-h v)) / 2h with f = <y, dy> summed in float64.  h = 2^-6: the third-order term is below
    h^2 ~ 2.5e-4 of the directional size, float32 noise ~ 1e-6 / h ~ 1e-4 of it."""
    g = torch.Generator().manual_seed(5)
    if op == "linear":
        leaves = [rand(60, 24, dtype=torch.float32, seed=1), rand(32, 24, dtype=torch.float32, seed=2, scale=0.2), rand(32, dtype=torch.float32, seed=3),
                  rand(60, 32, dtype=torch.float32, seed=4)]
        f = lambda x, w, b, r: geot.linear(x, w, b, residual=r, activation="gelu")  # noqa: E731
    elif op == "segment_matmul":
        ptr = torch.tensor([0, 10, 10, 60], device="cuda")
        leaves = [rand(60, 24, dtype=torch.float32, seed=1), rand(3, 24, 32, dtype=torch.float32, seed=2, scale=0.2), rand(3, 32, dtype=torch.float32, seed=3)]
        f = lambda x, w, b: geot.segment_matmul(x, ptr, w, b)  # noqa: E731
    else:
        leaves = [rand(60, 40, dtype=torch.float32, seed=1), rand(40, dtype=torch.float32, seed=2), rand(40, dtype=torch.float32, seed=3)]
        f = geot.layer_norm
    y = f(*[t.requires_grad_() for t in leaves])
    dy = torch.randn(y.shape, generator=g).cuda()
    grads = torch.autograd.grad(y, leaves, dy)
    h = 2.0 ** -6
    with torch.no_grad():
        for i, (leaf, grad) in enumerate(zip(leaves, grads)):
            v = torch.randn(leaf.shape, generator=g).cuda()
            up, down = ([t + s * h * v if j == i else t for j, t in enumerate(leaves)] for s in (1, -1))
            fd = float(((f(*up).double() - f(*down).double()) * dy.double()).sum()) / (2 * h)
            an = float((grad.double() * v.double()).sum())
            scale = float(grad.double().norm() * v.double().norm()) / math.sqrt(v.numel())
            assert abs(fd - an) <= 2e-3 * max(scale, abs(an)), (i, fd, an)


@gpu
def test_second_derivatives_are_refused():
    x, w = rand(8, 16, dtype=torch.float32, seed=1).requires_grad_(), rand(16, 16, dtype=torch.float32, seed=2).requires_grad_()
    ptr = torch.tensor([0, 8], device="cuda")
    for y in (geot.linear(x, w), geot.segment_matmul(x, ptr, w[None]), geot.layer_norm(x)):
        with pytest.raises(NotImplementedError, match="not differentiable"):
            torch.autograd.grad(y.sum(), [x], create_graph=True)


@gpu
def test_streams():
    """On a stream of their own, inputs produced there."""
    n, edges, rows, ptr, tensors = _typed_problem(3)
    want = _typed_layer(tensors[0], edges, ptr, *tensors[1:], n)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        x = tensors[0].clone()
        got = _typed_layer(x, edges, ptr, *tensors[1:], n)
    s.synchronize()
    assert torch.equal(got, want)


@gpu
def test_graph_capture():
    """Two captured graphs - inference, and forward with gradients - replayed in turn with eager work and new inputs between."""
    rows = [0, 100, 100, 5000, 9000]
    ptr = torch.tensor(rows, device="cuda")
    shapes = [((9000, 40), 1), ((4, 40, 72), 0.2), ((48, 72), 0.2), ((48,), 1), ((9000, 48), 1), ((48,), 1), ((48,), 1)]
    t = [rand(*s, dtype=torch.bfloat16, seed=i, scale=sc) for i, (s, sc) in enumerate(shapes)]
    dy = rand(9000, 48, dtype=torch.bfloat16, seed=50)

    def forward(x, wseg, w, b, r, gamma, beta):
        return geot.layer_norm(geot.linear(geot.segment_matmul(x, ptr, wseg), w, b, residual=r, activation="gelu"), gamma, beta)

    def train():
        leaves = [a.detach().requires_grad_() for a in t]
        y = forward(*leaves)
        return [y.detach(), *torch.autograd.grad(y, leaves, dy)]

    def infer():
        with torch.no_grad():
            return [forward(*t)]

    graphs, outs = [], []
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        infer(), train()
    torch.cuda.current_stream().wait_stream(s)
    for fn in (infer, train):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = fn()
        graphs.append(graph)
        outs.append(out)
    for turn in range(4):
        with torch.no_grad():
            for i, a in enumerate(t):
                a.copy_(rand(*a.shape, dtype=a.dtype, seed=1000 * (turn + 1) + i, scale=shapes[i][1]))
        want = [infer(), train()]
        for graph in (graphs if turn % 2 else graphs[::-1]):
            graph.replay()
        torch.cuda.synchronize()
        for w_, o_ in zip(want, outs):
            for a, c in zip(w_, o_):
                assert torch.equal(a, c)
        want = train()                               # (eager work between the replays)
        torch.cuda.synchronize()


@gpu
def test_compile():
    torch._dynamo.reset()
    n, edges, rows, ptr, tensors = _typed_problem(7)
    x, w, b = tensors[0], tensors[2], tensors[3]

    def f(x, w, b, gamma):
        h = geot.segment_matmul(geot.linear(x, w, b, activation="gelu"), ptr, tensors[1])
        return geot.layer_norm(h, gamma)

    ptr = torch.tensor([0, 10, 50, 50, 90, 200, 400], device="cuda")
    leaves = [a.detach().requires_grad_() for a in (x, w, b, tensors[4])]
    want = f(*leaves)
    grads = torch.autograd.grad(want.sum(), leaves)
    got = torch.compile(f)(*leaves)
    for a, c in zip((want, *grads), (got, *torch.autograd.grad(got.sum(), leaves))):
        assert torch.allclose(a, c, rtol=1e-5, atol=1e-5)
    with torch.no_grad():
        assert torch.allclose(torch.compile(f)(*leaves), want, rtol=1e-5, atol=1e-5)


# ---- in rewritten models ----------------------------------------------------------------------------------------------------------------
class _Block(torch.nn.Module):
    """A layer in plain torch: aggregation, feed-forward with a skip connection, normalisation, and a product that must keep its form."""

    def __init__(self, f):
        super().__init__()
        self.a, self.b, self.c = torch.nn.Linear(f, 2 * f), torch.nn.Linear(2 * f, f), torch.nn.Linear(f, f, bias=False)
        self.norm = torch.nn.LayerNorm(f)

    def forward(self, x, edge_index):
        row, col = edge_index[0], edge_index[1]
        agg = x.new_zeros(x.shape).index_add(0, row, x.index_select(0, col))
        h = self.b(torch.nn.functional.gelu(self.a(agg))) + x
        z = self.c(h)
        return self.norm(torch.nn.functional.silu(z)) * z       # z is used twice: its activation stays outside


def _block_problem(device):
    torch.manual_seed(0)
    g = torch.Generator().manual_seed(1)
    row = torch.sort(torch.randint(0, 300, (2000,), generator=g)).values
    return _Block(24).to(device), (torch.randn(300, 24, generator=g).to(device), torch.stack([row, torch.randint(0, 300, (2000,), generator=g)]).to(device))


def test_rewritten_model_nodes():
    from geot_amd.match_replace import pattern_transform
    model, args = _block_problem("cpu")
    plain = pattern_transform(model, args)
    assert plain.geot_dense_nodes == 0 and plain.geot_fused_nodes == 1
    ep = pattern_transform(model, args, dense=True)
    nodes = [n for n in ep.graph_module.graph.nodes if n.op == "call_function"]
    linears = [n for n in nodes if n.target == torch.ops.geot_dense.linear.default]
    assert ep.geot_dense_nodes == 4 and ep.geot_fused_nodes == 1
    assert [(n.args[4], n.args[3] is not None, n.args[2] is not None) for n in linears] == [("gelu", False, True), ("none", True, True), ("none", False, False)]
    assert sum(n.target == torch.ops.geot_dense.layer_norm.default for n in nodes) == 1
    assert sum(n.target == torch.ops.aten.silu.default for n in nodes) == 1


@gpu
def test_rewritten_model_computes_and_trains():
    from geot_amd.match_replace import pattern_transform
    model, args = _block_problem("cuda")
    want = model(*args)
    params = list(model.parameters())
    dy = torch.randn(want.shape, generator=torch.Generator().manual_seed(2)).cuda()
    grads = torch.autograd.grad(want, params, dy)
    ep = pattern_transform(model, args, dense=True)
    mod = ep.module()
    got = mod(*args)
    new = dict(mod.named_parameters())
    got_grads = torch.autograd.grad(got, [new[k] for k, _ in model.named_parameters()], dy)
    for a, b in zip((want, *grads), (got, *got_grads)):
        assert float((a - b).abs().max()) <= 1e-4 * max(1.0, float(a.abs().max()))
    with torch.no_grad():
        assert float((mod(*args) - want).abs().max()) <= 1e-4 * max(1.0, float(want.abs().max()))
