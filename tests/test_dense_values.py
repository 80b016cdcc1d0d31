"""linear, segment_matmul and layer_norm at values and on paths where single numbers matter: infinities, tails, masked places, every kernel.

Tolerances count roundings: u = half a step of the dtype, 2^-23 a step of a float32 sum.
"""
import math

import pytest
import torch

import geot_amd as geot
from test_dense_ops import LinearReference, close

gpu = pytest.mark.gpu
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
IDS = ["f32", "f16", "bf16"]
INF, NAN = float("inf"), float("nan")
# rows, in, out of a product and the kernel it takes: 128-row tiles, few rows (narrow: z computed again in the backward pass; wide: z
# kept), a reduction split over workgroups
PATHS = {"tile": (200, 64, 72), "few": (33, 128, 40), "few-kept": (20, 512, 40), "split": (100, 4160, 48)}


# ---- refusals: no GPU needed ----------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("device", ["cpu", "meta"])
def test_forward_mode_is_refused(device):
    """A tangent of any input, through dual tensors or torch.func, alone or beside reverse mode: named, never dropped."""
    import torch.autograd.forward_ad as forward_ad
    ones = lambda *s: torch.ones(*s, device=device)  # noqa: E731
    ptr = torch.tensor([0, 1, 4]).to(device)
    calls = {"linear": (lambda x, w, b, r: geot.linear(x, w, b, residual=r), [ones(4, 6), ones(5, 6), ones(5), ones(4, 5)]),
             "segment_matmul": (lambda x, w, b: geot.segment_matmul(x, ptr, w, b), [ones(4, 6), ones(2, 6, 5), ones(2, 5)]),
             "layer_norm": (geot.layer_norm, [ones(4, 6), ones(6), ones(6)])}
    for name, (f, args) in calls.items():
        for i, t in enumerate(args):
            one = lambda v: f(*args[:i], v, *args[i + 1:])  # noqa: E731, B023
            refused = pytest.raises(NotImplementedError, match=f"{name}: forward-mode gradients .* not supported")
            with refused, forward_ad.dual_level():
                one(forward_ad.make_dual(t, torch.ones_like(t)))
            with refused, forward_ad.dual_level():
                one(forward_ad.make_dual(t.clone().requires_grad_(), torch.ones_like(t)))
            with refused:
                torch.func.jvp(one, (t,), (torch.ones_like(t),))
            with refused, torch.no_grad():
                torch.func.jvp(one, (t,), (torch.ones_like(t),))
            with refused:
                torch.func.jacfwd(one)(t)


class _Writes(torch.nn.Module):
    """In-place operators between a product and what consumes it: on the product's input, its weight, the skip connection."""

    def __init__(self, where):
        super().__init__()
        self.lin, self.where = torch.nn.Linear(6, 6), where

    def forward(self, x):
        h = x * 2
        z = self.lin(h)
        if self.where == "activation":
            h.add_(1)
        y = torch.relu(z)
        if self.where == "addition":
            h.mul_(3)
        if self.where == "elsewhere":
            x = torch.zeros_like(x).view(-1)[:6] + x
        return y + h, x


@pytest.mark.parametrize("where,form", [("activation", ("none", False)), ("addition", ("relu", False)), ("elsewhere", ("relu", True))])
def test_rewriting_keeps_the_order_of_writes(where, form):
    """The fused node reads its operands where the last part of it stood: in front of no write that was there before."""
    from geot_amd.match_replace import pattern_transform
    torch.manual_seed(0)
    model, x = _Writes(where), torch.randn(4, 6)
    ep = pattern_transform(model, (x,), dense=True)
    nodes = [n for n in ep.graph_module.graph.nodes if n.target == torch.ops.geot_dense.linear.default]
    assert [(n.args[4], n.args[3] is not None) for n in nodes] == [form]

    def plain_linear(x, w, b, r, act):
        y = torch.nn.functional.linear(x, w, b)
        y = torch.relu(y) if act == "relu" else y
        return y if r is None else y + r

    nodes[0].target = plain_linear                       # (what the node computes, on the CPU)
    ep.graph_module.recompile()
    got = ep.graph_module(*[p.detach() for p in model.parameters()], x)
    for a, b in zip(got, model(x)):
        assert torch.equal(a, b.detach())


def test_impossible_sizes_are_refused():
    """Sizes whose products pass 64 bits: an error code, no division by zero on the way (in a process of its own: a signal would end it)."""
    import subprocess
    import sys
    code = """
import geot_amd as geot
L, big = geot._lib.load(), 1 << 40
for a, b, c in ((1, big, big), (big, big, 1), (big, 1, big), (big, big, big), (1 << 62, 1, 1), (-1, 4, 4)):
    for dtype in (0, 2, 3):
        assert L.geot_linear_workspace_bytes(a, b, c, dtype) == L.geot_linear_grad_input_workspace_bytes(a, b, c, dtype) == 0
        assert L.geot_linear_grad_weight_workspace_bytes(a, b, c, dtype) == 0
        assert L.geot_segment_matmul_workspace_bytes(a, 3, b, c, dtype) == L.geot_segment_matmul_grad_weight_workspace_bytes(a, 3, b, c, dtype) == 0
        assert L.geot_linear(16, b, 16, None, None, 0, None, 16, a, b, c, 0, dtype, None, 0, None) == -1
        assert L.geot_linear_grad_input(16, 16, 16, a, b, c, dtype, None, 0, None) == -1
        assert L.geot_linear_grad_weight(16, 16, b, 16, 16, a, b, c, dtype, 16, 1 << 62, None) == -1
        assert L.geot_segment_matmul(16, b, 16, 16, None, 16, a, 3, b, c, dtype, 16, 1 << 62, None) == -1
        assert L.geot_segment_matmul_grad_weight(16, b, 16, 16, 16, 16, a, 3, b, c, dtype, 16, 1 << 62, None) == -1
for rows, feat in ((1 << 62, 4), (big, 1 << 20), (4, 1 << 40), (-1, 4)):
    assert L.geot_layer_norm(16, feat, None, None, 16, None, rows, feat, 1e-5, 0, 0, None) == -1
    assert L.geot_layer_norm_backward_workspace_bytes(rows, feat) == 0
    assert L.geot_layer_norm_backward(16, feat, None, 16, 16, 16, None, None, rows, feat, 0, 0, None, 0, None) == -1
# one row, as many groups as there may be, a long reduction: its shares stay inside one launch (fewer than 2^32 threads)
need = L.geot_segment_matmul_workspace_bytes(1, 65535, 65536, 1, 2)
assert 0 < need <= ((1 << 32) // (256 * 65537)) * 4, need
print("refused")
"""
    p = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, cwd=geot._lib._ROOT)
    assert p.returncode == 0 and p.stdout.strip() == "refused", (p.returncode, p.stdout, p.stderr[-500:])


def test_segment_workspace_does_not_grow_with_groups():
    """Only chunks of groups that have several need room: at fixed rows no number of groups asks for more than twice the chunks of all rows."""
    L = geot._lib.load()
    one = (64 * 128 + 128) * 4
    for rows in (1, 256, 257, 20_000, 1_000_003):
        for dtype in (0, 2, 3):
            sizes = [L.geot_segment_matmul_grad_weight_workspace_bytes(rows, groups, 64, 128, dtype) for groups in (1, 16, 256, 4096, 65535)]
            assert max(sizes) <= 2 * -(-rows // 256) * one and sizes[-1] == sizes[-2], (rows, dtype, sizes)
    # 256 groups of 4096 x 4096 and 20,000 rows: two chunks of 16384 rows, of which one group could have both
    need = L.geot_segment_matmul_grad_weight_workspace_bytes(20_000, 256, 4096, 4096, 2)
    assert need <= 4 * (4096 * 4096 + 4096) * 4


@pytest.mark.parametrize("where", ["nowhere", "rows", "factor", "factor, copied before", "zeros", "row of zeros"])
def test_rewriting_an_aggregation_keeps_the_order_of_writes(where):
    from geot_amd.match_replace import pattern_transform

    class Aggregate(torch.nn.Module):
        def forward(self, x, w, row, col):
            h, f = x * 2, w * 2
            column = f.unsqueeze(-1)
            if where.startswith("factor,"):
                column = column.clone()
                f.add_(1)
            rows = h.index_select(0, col)
            out = h.new_zeros(5, 6)
            scaled = column * rows
            if where in ("rows", "factor", "zeros", "row of zeros"):
                {"rows": h, "factor": f, "zeros": out, "row of zeros": out[0]}[where].add_(1)
            return out.index_add(0, row, scaled) + h.sum() + f.sum()

    row = torch.tensor([0, 1, 1, 3])
    ep = pattern_transform(Aggregate(), (torch.randn(5, 6), torch.randn(4), row, row))
    assert ep.geot_fused_nodes == (where == "nowhere")


def test_rewriting_a_model_on_the_cpu_warns():
    import warnings
    from geot_amd.match_replace import pattern_transform
    args = (torch.randn(4, 6),)
    with pytest.warns(UserWarning, match="run on the GPU only"):
        pattern_transform(torch.nn.Linear(6, 6), args, dense=True)
    with warnings.catch_warnings():
        warnings.filterwarnings("error", message=".*run on the GPU only")
        pattern_transform(torch.nn.Linear(6, 6), args)                               # (nothing rewritten, nothing to say)
        pattern_transform(torch.nn.Linear(6, 6).double(), (args[0].double(),), dense=True)


# ---- activations ----------------------------------------------------------------------------------------------------------------------
def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def normal_cdf(z):
    return torch.special.erfc(z * -math.sqrt(0.5)) / 2       # (torch.special.ndtr is 1 + erf on the GPU: 0 below -8.3)


def act64(z, name):
    if name == "relu":
        return torch.relu(z)
    return z * (normal_cdf(z) if name == "gelu" else torch.sigmoid(z)) if name != "none" else z


def slope64(z, name):
    """With the limits 0 and 1 at the infinities."""
    c = z.clamp(-1000, 1000)
    if name == "relu":
        s = (z > 0).double()
    elif name == "gelu":
        s = normal_cdf(c) + c * torch.exp(-c * c / 2) / math.sqrt(2 * math.pi)
    else:
        s = torch.sigmoid(c) * (1 + c * torch.sigmoid(-c))
    return torch.where(torch.isnan(z), z, s)


def through_linear(z, path, act):
    """act(z) and act'(z) of a column of values that the product hands through unchanged: one weight is 1 (two, where z is a pair's sum),
    the rest is 0, and one output's gradient is 1."""
    m, k, n = PATHS[path]
    rows = z.shape[0]
    x = torch.zeros(m, k, dtype=z.dtype, device=z.device)
    x[:rows, :z.shape[1]] = z
    w = torch.zeros(n, k, dtype=z.dtype, device=z.device)
    w[:, :z.shape[1]] = 1
    with torch.no_grad():
        y = geot.linear(x, w, activation=act)
    x.requires_grad_()
    yt = geot.linear(x, w, activation=act)
    assert torch.equal(yt.nan_to_num(7.0), y.nan_to_num(7.0))
    dy = torch.zeros(m, n, dtype=z.dtype, device=z.device)
    dy[:, 3] = 1
    (dx,) = torch.autograd.grad(yt, [x], dy)
    assert bool((y[:rows] == y[:rows, :1]).logical_or(torch.isnan(y[:rows, :1])).all())
    return y[:rows, 0], dx[:rows, 0]


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("path", PATHS)
@pytest.mark.parametrize("act", ["relu", "gelu", "silu"])
def test_activations_at_infinities(act, path, dtype):
    """Infinities, NaN and sums that pass the dtype's range: values as the formula gives them, slopes by their limits."""
    big = 60000.0 if dtype == torch.float16 else 1e38
    pairs = [(INF, 0), (-INF, 0), (NAN, 0), (0.0, 0), (2, 0), (-2, 0), (30, 0), (-30, 0), (1e4, 0), (-1e4, 0), (big, 0), (-big, 0), (big, big), (-big, -big)]
    z = torch.tensor(pairs, dtype=dtype, device="cuda")
    y, slope = through_linear(z, path, act)
    total = z.double().sum(1)
    want = act64(total, act)
    over = want.abs() > torch.finfo(dtype).max               # (rounds to an infinity)
    want = torch.where(over, want.sign() * INF, want)
    assert torch.equal(torch.isnan(y), torch.isnan(want)) and torch.equal(torch.isinf(y), torch.isinf(want)), (y, want)
    fine = torch.isfinite(want)
    tol = (half_step(dtype) + 2.0 ** -15) * want.abs() + torch.finfo(dtype).tiny
    assert bool(((y.double() - want).abs() <= tol)[fine].all()), (y, want)
    want = slope64(total, act)
    assert torch.equal(torch.isnan(slope), torch.isnan(want)), (slope, want)
    tol = half_step(dtype) * want.abs() + 2.0 ** -15
    assert bool(((slope.double() - want).abs() <= tol)[~torch.isnan(want)].all()), (slope, want)


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("path", ["tile", "few-kept"])
@pytest.mark.parametrize("act", ["gelu", "silu"])
def test_activation_tails(act, path, dtype):
    """Values and slopes from -14 to 14, relative to their size.  What a form may be off beside the rounding of its result:
    float32 gelu: 4e-7 of the tail is its fit, the exponent's products (up to 2^7 of 2^-24 each) the rest: 2^-19; slopes and silu alike.
    16-bit gelu: 2^-13 of the tail (fits 2^-17 and 2^-15 up to 10, float32 rounding of the exponent behind); slopes 2^-15.  silu in 16 bits
    rounds z log2(e) once: 14 * 1.45 * 2^-24 * ln 2 = 2^-20.  A float16 result is rounded to half a subnormal step at least; in the
    other types results below the smallest normal number, and a tail below 2^-126 times 14, may be 0.  Around the zero of gelu's slope (-0.75) the terms that cancel there are of size 0.3."""
    rows = PATHS[path][0]
    z = torch.cat([torch.linspace(-14, 14, rows - 4), torch.tensor([-0.75, -0.7518, -12.75, 5.8])])[:rows].to(dtype).cuda()
    y, slope = through_linear(z[:, None], path, act)
    z = z.double()
    fit = {"gelu": 2.0 ** -19 if dtype == torch.float32 else 2.0 ** -13, "silu": 2.0 ** -19}[act]
    tiny = 2.0 ** -25 if dtype == torch.float16 else 15 * 2.0 ** -126
    want = act64(z, act)
    tail = want - z.clamp(min=0)                             # what is computed beside max(z, 0), which is exact
    tol = half_step(dtype) * want.abs() + 2.0 ** -22 * want.abs() + fit * tail.abs() + tiny
    off = (y.double() - want).abs() > tol
    assert not off.any(), (z[off], y[off], want[off])
    want = slope64(z, act)
    fit = 2.0 ** -19 if dtype == torch.float32 else 2.0 ** -15
    size = torch.minimum(want.abs(), (1 - want).abs()) + 0.3 * ((z.abs() > 0.3) & (z.abs() < 1.6))
    if act == "silu":                                        # s (1 + z (1 - s)): its bracket cancels at -1.28, as large as the two terms together
        size = torch.sigmoid(z) * (1 + z.abs() * torch.sigmoid(-z))
    tol = half_step(dtype) * want.abs() + 2.0 ** -22 * want.abs() + fit * size + tiny
    off = (slope.double() - want).abs() > tol
    assert not off.any(), (z[off], slope[off], want[off])


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("path", PATHS)
@pytest.mark.parametrize("residual", [False, True], ids=["plain", "skip"])
def test_relu_keeps_masked_gradients_out(residual, path, dtype):
    """An infinite or NaN gradient where relu is off reaches nothing but the residual: dx and db are what they are with 0 there."""
    m, k, n = PATHS[path]
    g = torch.Generator().manual_seed(1)
    x, w, b, r, dy = (torch.randn(*s, generator=g).to(dtype).cuda() for s in ((m, k), (n, k), (n,), (m, n), (m, n)))
    w[5:9] = 0
    b[5:8] = torch.tensor([-1.0, 0.0, -3.0])
    leaves = [t.requires_grad_() for t in (x, w, b)] + ([r.requires_grad_()] if residual else [])

    def grads(dy):
        return torch.autograd.grad(geot.linear(x, w, b, residual=r if residual else None, activation="relu"), leaves, dy)

    clean, dirty = dy.clone(), dy.clone()
    clean[:, 5:8] = 0
    dirty[:, 5:8] = torch.tensor([INF, NAN, -INF], dtype=dtype)
    got = grads(dirty)
    for a, c in zip(got[:3], grads(clean)[:3]):
        assert torch.equal(a, c)
    if residual:
        assert torch.equal(got[3].nan_to_num(7.0), dirty.nan_to_num(7.0))


# ---- every kernel -----------------------------------------------------------------------------------------------------------------------
@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_segment_gradients_of_chunked_groups(dtype):
    """Groups of one to three chunks of 256 rows beside empty and tiny ones, ends on, before and behind a chunk's border, more groups than
    chunks: dW and db of every group, twice, bit for bit.  Integers of at most 4 and sums below 2^11 come out exactly in every type."""
    sizes = [0, 257, 1, 512, 0, 0, 513, 3, 256, 255, 700, 0, 2, 300, 1, 258, 511, 0, 0, 0, 769, 5] + [0, 1] * 20
    rows = [0]
    for s in sizes:
        rows.append(rows[-1] + s)
    k, n, m = 20, 72, rows[-1] + 9
    g = torch.Generator().manual_seed(3)
    x, dy = (torch.randint(-1, 2, s, generator=g).to(dtype).cuda() for s in ((m, k), (m, n)))
    w, b = torch.zeros(len(sizes), k, n, dtype=dtype, device="cuda", requires_grad=True), torch.zeros(len(sizes), n, dtype=dtype, device="cuda", requires_grad=True)
    ptr = torch.tensor(rows, device="cuda")
    runs = [torch.autograd.grad(geot.segment_matmul(x, ptr, w, b), [w, b], dy) for _ in range(2)]
    for i in range(len(sizes)):
        lo, hi = rows[i], rows[i + 1]
        dw, db = x[lo:hi].double().t().contiguous() @ dy[lo:hi].double(), dy[lo:hi].double().sum(0)
        for run in runs:
            # (bfloat16 holds whole numbers up to 256; sums of 769 numbers of -1, 0, 1 stay below: 6 standard deviations are 150)
            assert torch.equal(run[0][i].double(), dw) and torch.equal(run[1][i].double(), db), i


@gpu
@pytest.mark.parametrize("m,k,n", [(200, 200, 72), (33, 300, 40), (100, 4160, 48), (1500, 70, 130)], ids=["tile", "few", "split", "chunks"])
def test_nonfinite_sums_of_long_reductions(m, k, n):
    """float32 sums that end in an infinity or NaN, decided by terms far behind the first: y, dx and dW of linear and segment_matmul have
    them where float64 arithmetic has, and everything else within the products' bound (6 partial products of 2^-23 steps a term).  Left
    out: sums whose finite terms pass float32's range in absolute value, of both signs or beside an infinity - a term or a partial sum
    becomes an infinity of either sign in float32 arithmetic, and it ends in an infinity, NaN or a number as its order has it."""
    g = torch.Generator().manual_seed(m)
    x, w, dy = (torch.randn(*s, generator=g).cuda() for s in ((m, k), (n, k), (m, n)))
    x[3, k - 2], x[5, 1], x[5, k - 1], x[m - 1, k // 2] = INF, INF, -INF, NAN
    w[n - 1, 2], w[1, k - 3] = -INF, NAN
    dy[m - 2, n - 2], dy[m // 2, 0], dy[0, 5], dy[m - 3, 5] = INF, NAN, 3e38, 3e38
    x[0, 0], x[m - 3, 0] = 2.0, 2.0                          # (dW[5, 0]: 2 * 3e38 twice)
    ptr = torch.tensor([0, m], device="cuda")

    def check(got, a, b, what):
        want, most = a.double() @ b.double(), torch.finfo(torch.float32).max
        size = a.double().nan_to_num(0, 0, 0).abs() @ b.double().nan_to_num(0, 0, 0).abs()
        open_ended = (size > most) & (torch.isinf(want) | (torch.isfinite(want) & (want.abs() < 0.99 * size)))
        want = torch.where(want.abs() > most, want.sign() * INF, want)
        got, want, size = got.double()[~open_ended], want[~open_ended], size[~open_ended]
        assert torch.equal(torch.isnan(got), torch.isnan(want)), what
        assert torch.equal(got[torch.isinf(want)], want[torch.isinf(want)]) and torch.equal(torch.isinf(got), torch.isinf(want)), what
        off = (got - want).abs() > (6 * a.shape[1] + 16) * 2.0 ** -23 * size
        assert not (off & torch.isfinite(want)).any(), what

    xg, wg, w3 = x.clone().requires_grad_(), w.clone().requires_grad_(), w.t()[None].contiguous().requires_grad_()
    for y, weight, flip in ((geot.linear(xg, wg), wg, False), (geot.segment_matmul(xg, ptr, w3), w3, True)):
        dx, dw = torch.autograd.grad(y, [xg, weight], dy)
        check(y, x, w.t().contiguous(), "y")
        check(dx, dy, w, "dx")
        check(dw[0].t() if flip else dw, dy.t().contiguous(), x, "dw")


def relative_error(got, want):
    return float((got.double() - want).norm() / want.norm())


@gpu
@pytest.mark.parametrize("dtype", DTYPES[1:], ids=IDS[1:])
@pytest.mark.parametrize("act", ["none", "relu", "gelu", "silu"])
@pytest.mark.parametrize("k", [128, 512], ids=["recomputed", "kept"])
def test_roundings_of_a_training_step(k, act, dtype):
    """How often the results of a 16-bit training step are rounded, by their error in 2-norm.  One rounding is uniform in half a step, at most
    eps / sqrt(12) of the value in root mean square.  y and db: one.  dx and dW: one more of dz if there is an activation; where z is kept, its
    own reaches dz through the slope's slope, at most 0.8 (gelu) or 0.5 (silu) times |z| eps / sqrt(12) against a slope of 0.5 or more in root
    mean square, |z| of size 1.  Fits, float32 sums and float16's subnormals: 2 % more."""
    m, n = 3000, 256
    g = torch.Generator().manual_seed(k)
    x, w, b, dy = ((torch.randn(*s, generator=g) * c).to(dtype).cuda() for s, c in (((m, k), 1), ((n, k), k ** -0.5), ((n,), 0.1), ((m, n), 1)))
    leaves = [t.requires_grad_() for t in (x, w, b)]
    y = geot.linear(*leaves, activation=act)
    dx, dw, db = torch.autograd.grad(y, leaves, dy)
    z = x.double() @ w.double().t().contiguous() + b.double()
    dz = dy.double() * (slope64(z, act) if act != "none" else 1)
    if act == "relu":                                        # (where float32 sums decide the sign)
        dz = torch.where(z.abs() < 1e-4, dy.double() * (y > 0), dz)
    one = torch.finfo(dtype).eps / math.sqrt(12)
    kept = {"gelu": 0.8, "silu": 0.5}.get(act, 0) / 0.5 if k == 512 else 0
    many = math.sqrt(1 + (act != "none") + kept ** 2) * one
    assert relative_error(y, act64(z, act)) <= 1.02 * one
    assert relative_error(db, dz.sum(0)) <= 1.02 * math.sqrt(1 + kept ** 2) * one
    assert relative_error(dx, dz @ w.double()) <= 1.02 * many
    assert relative_error(dw, dz.t().contiguous() @ x.double()) <= 1.02 * many


def _edges_of_tiles(m, tile=256):
    """Rows to look at: ends of the first and last tiles, both sides of their borders, some between."""
    g = torch.Generator().manual_seed(m)
    last = m // tile * tile
    near = [0, 1, 31, 127, 128, tile - 1, tile, tile + 1, 2 * tile - 1, last - 1]
    return torch.cat([torch.tensor(near), torch.randint(0, m, (60,), generator=g), torch.arange(last, m)]).unique().cuda()


# 16-bit rows and 512 or more values a sum: 256 x 256 tiles, two buffers; reductions of whole steps of 64 and not, odd and even in number
WIDE = [(66_001, 602, 258), (66_000, 520, 300), (66_301, 576, 256), (66_000, 640, 511)]


@gpu
@pytest.mark.parametrize("dtype", DTYPES[1:], ids=IDS[1:])
@pytest.mark.parametrize("m,k,n", WIDE)
def test_linear_in_large_tiles(m, k, n, dtype):
    g = torch.Generator(device="cuda").manual_seed(k)
    x, r = (torch.randn(m, c, generator=g, device="cuda").to(dtype) for c in (k, n))
    w, b = (torch.randn(n, k, generator=g, device="cuda") * k ** -0.5).to(dtype), torch.randn(n, generator=g, device="cuda").to(dtype)
    rows = _edges_of_tiles(m)
    one = 1.02 * torch.finfo(dtype).eps / math.sqrt(12)
    kind = {torch.float16: "_Float16", torch.bfloat16: "__bf16"}[dtype]
    for act, bias, res in (("none", None, None), ("gelu", b, r)):
        y = geot.linear(x, w, bias, residual=res, activation=act)
        assert geot.hip.last_kernel() == f"mm_rows_kernel<{kind}, 256, 256, 2, 4, false, 2, false>"
        ref = LinearReference(x[rows], w, bias, None if res is None else r[rows], act)
        close(y[rows], ref.y, ref.e_y, f"y {act}")
        assert relative_error(y[rows], ref.y) <= one
        whole = torch.nn.functional.linear(x, w, bias)       # (every row: no tile left out or written twice; another library's rounding beside)
        whole = whole if act == "none" else torch.nn.functional.gelu(whole) + r
        assert float((y.float() - whole.float()).abs().max()) <= 8 * torch.finfo(dtype).eps * float(whole.float().abs().max())
    # the gradient of the input, where the weight's output index is contiguous
    w2 = (torch.randn(k, n, generator=g, device="cuda") * k ** -0.5).to(dtype)
    x2 = torch.zeros(m, n, dtype=dtype, device="cuda")
    dx = torch.ops.geot_dense.linear_backward(x, x2, w2, None, x2[:0, 0], "none", True, False, False)[0]    # (in this thread, for last_kernel)
    assert geot.hip.last_kernel() == f"mm_rows_kernel<{kind}, 256, 256, 2, 4, true, 2, false>"
    ref = LinearReference(x[rows], w2.t(), None, None, "none")
    close(dx[rows], ref.y, ref.e_y, "dx")
    assert relative_error(dx[rows], ref.y) <= one
    whole = x.float() @ w2.float()
    assert float((dx.float() - whole).abs().max()) <= 8 * torch.finfo(dtype).eps * float(whole.abs().max())


@gpu
@pytest.mark.parametrize("dtype", DTYPES[1:], ids=IDS[1:])
def test_segment_matmul_in_large_tiles(dtype):
    """Two groups above 2048 rows and an odd border, rows in front of and behind them: both directions in 256 x 256 tiles."""
    m, k, n, ptr = 66_000, 520, 602, [3, 30_001, 65_990]
    g = torch.Generator(device="cuda").manual_seed(1)
    x, dy = (torch.randn(m, c, generator=g, device="cuda").to(dtype) for c in (k, n))
    w = (torch.randn(2, k, n, generator=g, device="cuda") * k ** -0.5).to(dtype)
    at = torch.tensor(ptr, device="cuda")
    y = geot.segment_matmul(x, at, w)
    kind = {torch.float16: "_Float16", torch.bfloat16: "__bf16"}[dtype]
    assert geot.hip.last_kernel() == f"mm_rows_kernel<{kind}, 256, 256, 2, 4, true, 2, false>"
    dx = torch.ops.geot_dense.segment_matmul_backward(dy, x, at, w, True, False, False)[0]
    assert geot.hip.last_kernel() == f"mm_rows_kernel<{kind}, 256, 256, 2, 4, false, 2, false>"
    for got in (y, dx):
        assert not got[:3].any() and not got[65_990:].any()
    one = 1.02 * torch.finfo(dtype).eps / math.sqrt(12)
    for i, (lo, hi) in enumerate(zip(ptr[:-1], ptr[1:])):
        rows = _edges_of_tiles(hi - lo) + lo
        for got, a, b in ((y, x, w[i].t()), (dx, dy, w[i])):
            ref = LinearReference(a[rows], b, None, None, "none")
            close(got[rows], ref.y, ref.e_y, "y" if got is y else "dx")
            assert relative_error(got[rows], ref.y) <= one
            whole = a[lo:hi].float() @ b.float().t()
            assert float((got[lo:hi].float() - whole).abs().max()) <= 8 * torch.finfo(dtype).eps * float(whole.abs().max())


# ---- float32 products: 24 bits on every path, errors in root mean square -------------------------------------------------------------------
def _numbers(*shape, seed):
    """Significands of 24 random bits, exponents spread over 2^-40 .. 2^40."""
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * 2.0 ** torch.randint(-40, 41, shape, generator=g)).cuda()


def _ones_and_numbers(n, seed):
    v = _numbers(n, seed=seed)
    v[::3] = -0.125
    return v


def _last_place(got, want):
    """A product of two 24-bit significands: half a step of its rounding, 2^-23 left out of the split product, a step of the sums it passes."""
    off = (got.double() - want).abs() > 2.0 ** -21.5 * want.abs()
    assert got.shape == want.shape and not off.any(), (got[off], want[off])


# rows, in, out: one and many rows, tiles, few rows (one and two row fragments), a split reduction
SELECT = [(1, 256, 40), (20, 640, 72), (70, 300, 33), (200, 96, 96), (100, 4160, 48), (300, 64, 200)]


@gpu
@pytest.mark.parametrize("m,k,n", SELECT)
def test_float32_keeps_24_bits_forward_and_dx(m, k, n):
    """One entry a row of the weight: every result is one product."""
    x, w = _numbers(m, k, seed=m), torch.zeros(n, k, device="cuda")
    at = torch.randint(0, k, (n,), generator=torch.Generator().manual_seed(n)).cuda()
    v = _ones_and_numbers(n, 3)
    w[torch.arange(n, device="cuda"), at] = v
    want = x.double()[:, at] * v.double()
    ptr = torch.tensor([0, m // 3, m], device="cuda")
    _last_place(geot.linear(x, w), want)
    _last_place(geot.segment_matmul(x, ptr, torch.stack([w.t(), w.t()])), want)
    # dx = dy W with W [k, n] of one entry a column: the same products
    dy, empty = x, torch.empty(0, device="cuda")
    w2 = w.t().contiguous()
    dx = torch.ops.geot_dense.linear_backward(dy, torch.zeros(m, n, device="cuda"), w2, None, empty, "none", True, False, False)[0]
    _last_place(dx, want)
    dx = torch.ops.geot_dense.segment_matmul_backward(dy, torch.zeros(m, n, device="cuda"), ptr, torch.stack([w, w]), True, False, False)[0]
    _last_place(dx, want)


@gpu
@pytest.mark.parametrize("m,k,n", [(1, 5, 7), (100, 64, 64), (2000, 48, 130), (5000, 130, 48), (1500, 70, 64), (900, 200, 300)])
def test_float32_keeps_24_bits_dw(m, k, n):
    """One row with an entry for every output: dW is one product each, in one of several chunks of rows."""
    x, dy = _numbers(m, k, seed=m), torch.zeros(m, n, device="cuda")
    at = torch.randint(0, m, (n,), generator=torch.Generator().manual_seed(n)).cuda()
    v = _ones_and_numbers(n, 4)
    dy[at, torch.arange(n, device="cuda")] = v
    want = v.double()[:, None] * x.double()[at]
    dw, db = torch.ops.geot_dense.linear_backward(dy, x, torch.zeros(n, k, device="cuda"), torch.zeros(n, device="cuda"), torch.empty(0, device="cuda"), "none",
                                                  False, True, True)[1:]
    _last_place(dw, want)
    assert torch.equal(db, v)
    ptr = torch.tensor([0, 0, m, m], device="cuda")
    dw, db = torch.ops.geot_dense.segment_matmul_backward(dy, x, ptr, torch.zeros(3, k, n, device="cuda"), False, True, True)[1:]
    _last_place(dw[1].t(), want)
    assert torch.equal(db[1], v) and not dw[[0, 2]].any() and not db[[0, 2]].any()


@gpu
def test_float32_keeps_24_bits_where_z_is_computed_again():
    """dz = dy silu'(z) with z = one product: the slope (2^-20 of its size, see above) of a z that lost its third part, 2^-17 of it, shows."""
    m, k = 400, 96
    g = torch.Generator().manual_seed(5)
    x, w = (3 * torch.randn(m, k, generator=g)).cuda(), torch.zeros(k, k, device="cuda")
    v = (torch.rand(k, generator=g) + 0.5).cuda()
    w[torch.arange(k, device="cuda"), torch.randperm(k, generator=g).cuda()] = v
    x.requires_grad_()
    y = geot.linear(x, w, activation="silu")
    (dx,) = torch.autograd.grad(y, [x], torch.ones_like(y))
    z = x.detach().double() @ w.double().t().contiguous()
    dz = slope64(z, "silu")
    assert relative_error(dx, dz @ w.double()) <= 2.0 ** -21
    assert relative_error(y, act64(z, "silu")) <= 2.0 ** -21


def rms_bound(k):
    """Of a float32 product's error over its size, both in root mean square: the long sum rounds once for 16 to 64 values of the reduction (a
    random walk, every step at most 2^-23 of the sum so far), in between 6 to 24 matrix instructions may truncate, which shrinks a sum by up
    to 2^-24 each, half of it on average.  Without an operand's third part it is 2^-18.8 and more."""
    return (12 + 2 * math.sqrt(k / 32)) * 2.0 ** -24


@gpu
@pytest.mark.parametrize("m,k,n", [(1, 256, 512), (20, 520, 200), (70, 1000, 130), (300, 200, 96), (300, 1000, 72), (100, 4160, 48), (1000, 64, 64)])
def test_float32_errors_in_root_mean_square(m, k, n):
    g = torch.Generator().manual_seed(m + k + n)
    x, w, dy = (torch.randn(*s, generator=g).cuda() for s in ((m, k), (n, k), (m, n)))
    ptr = torch.tensor([0, m], device="cuda")
    x.requires_grad_()
    for weight, f in ((w.clone().requires_grad_(), geot.linear), (w.t()[None].contiguous().requires_grad_(), lambda x, w: geot.segment_matmul(x, ptr, w))):
        y = f(x, weight)
        dx, dw = torch.autograd.grad(y, [x, weight], dy)
        x64, w64, dy64 = x.detach().double(), w.double(), dy.double()
        assert relative_error(y, x64 @ w64.t().contiguous()) <= rms_bound(k)
        assert relative_error(dx, dy64 @ w64) <= rms_bound(n)
        assert relative_error(dw if dw.dim() == 2 else dw[0].t(), dy64.t().contiguous() @ x64) <= rms_bound(m)


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_many_rows_in_root_mean_square(dtype):
    """Sums over 70,001 rows: a row left out is 1 / sqrt(70001) = 2^-8 of dW and db, a chunk 2^-4; the bounds are one rounding of the
    result and the sums' own (float32: rms_bound of all rows)."""
    m, k, n = 70_001, 40, 24
    g = torch.Generator().manual_seed(9)
    x, dy = (torch.randn(m, c, generator=g).to(dtype).cuda() for c in (k, n))
    bound = rms_bound(m) if dtype == torch.float32 else 1.02 * torch.finfo(dtype).eps / math.sqrt(12)
    w, b = torch.zeros(n, k, dtype=dtype, device="cuda", requires_grad=True), torch.zeros(n, dtype=dtype, device="cuda", requires_grad=True)
    dw, db = torch.autograd.grad(geot.linear(x, w, b), [w, b], dy)
    assert relative_error(dw, dy.double().t().contiguous() @ x.double()) <= bound
    assert relative_error(db, dy.double().sum(0)) <= bound
    # relu at z = 0.5: dz = dy through the activation's own column sums
    half = torch.full((n,), 0.5, dtype=dtype, device="cuda", requires_grad=True)
    dw, db = torch.autograd.grad(geot.linear(x, w, half, activation="relu"), [w, half], dy)
    assert relative_error(dw, dy.double().t().contiguous() @ x.double()) <= bound
    assert relative_error(db, dy.double().sum(0)) <= bound
    ptr = torch.tensor([1, 30_000, 30_000, 70_000], device="cuda")
    w3, b3 = torch.zeros(3, k, n, dtype=dtype, device="cuda", requires_grad=True), torch.zeros(3, n, dtype=dtype, device="cuda", requires_grad=True)
    dw, db = torch.autograd.grad(geot.segment_matmul(x, ptr, w3, b3), [w3, b3], dy)
    for i, (lo, hi) in enumerate(((1, 30_000), (30_000, 30_000), (30_000, 70_000))):
        if lo == hi:
            assert not dw[i].any() and not db[i].any()
            continue
        assert relative_error(dw[i], x[lo:hi].double().t().contiguous() @ dy[lo:hi].double()) <= bound
        assert relative_error(db[i], dy[lo:hi].double().sum(0)) <= bound


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("m,d", [(60_011, 24), (3001, 602), (501, 2100), (401, 5000), (301, 9000)])
def test_layer_norm_in_root_mean_square(m, d, dtype):
    """y, dx, dw and db: one rounding of the result, and float32 sums of the row (at most 2 sqrt(d / 256) + 12 roundings of 2^-24) and over the
    rows (as many per partial row, then their join): 64 * 2^-24 holds all.  A row left out of dw or db is 1 / sqrt(m): 2^-8 and more."""
    g = torch.Generator().manual_seed(d)
    x, dy, w, b = (torch.randn(*s, generator=g).to(dtype).cuda().requires_grad_() for s in ((m, d), (m, d), (d,), (d,)))
    bound = 64 * 2.0 ** -24 + (0 if dtype == torch.float32 else 1.02 * torch.finfo(dtype).eps / math.sqrt(12))
    y = geot.layer_norm(x, w, b)
    dx, dw, db = torch.autograd.grad(y, [x, w, b], dy.detach())
    x64, dy64, w64, b64 = (t.detach().double() for t in (x, dy, w, b))
    var, mean = torch.var_mean(x64, -1, unbiased=False, keepdim=True)
    s = (var + 1e-5).rsqrt()
    h = (x64 - mean) * s
    gw = dy64 * w64
    assert relative_error(y, h * w64 + b64) <= bound
    assert relative_error(dx, s * (gw - gw.mean(-1, keepdim=True) - h * (gw * h).mean(-1, keepdim=True))) <= bound
    assert relative_error(dw, (dy64 * h).sum(0)) <= bound
    assert relative_error(db, dy64.sum(0)) <= bound


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("d", [16, 100, 300, 1500, 3000, 5000, 9000])
def test_layer_norm_parameter_gradients_alone(d, dtype):
    """The rows need no gradient: none is made, and the parameters' are the same bits."""
    g = torch.Generator().manual_seed(d)
    x, dy, w, b = (torch.randn(*s, generator=g).to(dtype).cuda() for s in ((37, d), (37, d), (d,), (d,)))
    w.requires_grad_(), b.requires_grad_()
    alone = torch.autograd.grad(geot.layer_norm(x, w, b), [w, b], dy)
    xg = x.clone().requires_grad_()
    dx, *both = torch.autograd.grad(geot.layer_norm(xg, w, b), [xg, w, b], dy)
    assert all(torch.equal(a, c) for a, c in zip(alone, both)) and bool(dx.any())
    stats = torch.ops.geot_dense.layer_norm_train(x, w, b, 1e-5)[1]
    none, dw, db = torch.ops.geot_dense.layer_norm_backward(dy, x, w, b, stats, False, True)
    assert none.numel() == 0 and torch.equal(dw, alone[0]) and torch.equal(db, alone[1])
    dx2, dw, db = torch.ops.geot_dense.layer_norm_backward(dy, x, w, b, stats, True, False)
    assert torch.equal(dx2, dx) and dw.numel() == db.numel() == 0


# ---- several at once --------------------------------------------------------------------------------------------------------------------
def _training_step(path, dtype, seed):
    m, k, n = PATHS[path]
    g = torch.Generator().manual_seed(seed)
    x, w, b, dy = ((torch.randn(*s, generator=g) * c).to(dtype).cuda() for s, c in (((m, k), 1), ((n, k), k ** -0.5), ((n,), 1), ((m, n), 1)))
    ptr = torch.tensor([0, m // 2, m], device="cuda")
    w3 = torch.stack([w.t(), w.t() * 0.5]).contiguous()
    inputs = [x, w, b, w3]

    def step():
        leaves = [t.detach().requires_grad_() for t in inputs]
        y = geot.layer_norm(geot.linear(*leaves[:3], activation="gelu"))
        z = geot.segment_matmul(leaves[0], ptr, leaves[3])
        return [y.detach(), z.detach(), *torch.autograd.grad([y, z], leaves, [dy, dy])]

    return inputs, step


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_two_threads_on_their_own_streams(dtype):
    """Training steps of every path from two threads at once: the bits of each step alone."""
    import threading
    steps = [_training_step(path, dtype, i)[1] for i, path in enumerate(PATHS)]
    want = [step() for step in steps]
    torch.cuda.synchronize()
    errors, done = [], []

    def work(order):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for _ in range(5):
                    for i in order:
                        for a, c in zip(steps[i](), want[i]):
                            if not torch.equal(a, c):
                                errors.append(i)
            stream.synchronize()
            done.append(True)
        except Exception as e:  # noqa: BLE001
            errors.append(repr(e))

    threads = [threading.Thread(target=work, args=(order,)) for order in ((0, 1, 2, 3), (3, 1, 0, 2))]
    for t in threads:
        t.start()
    for t in threads:
        t.join(timeout=60)
    assert not errors and len(done) == 2, errors


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
def test_every_path_in_two_captured_graphs(dtype):
    """Each path's training step in two graphs with scratch of their own, replayed in turn on new inputs with eager steps between."""
    for i, path in enumerate(PATHS):
        pair = [_training_step(path, dtype, 10 * i + j) for j in range(2)]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            for _, step in pair:
                step()
        torch.cuda.current_stream().wait_stream(side)
        graphs, outs = [], []
        for _, step in pair:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                outs.append(step())
            graphs.append(graph)
        for turn in range(3):
            g = torch.Generator(device="cuda").manual_seed(turn)
            for inputs, _ in pair:
                for t in inputs:
                    t.copy_(torch.randn(t.shape, generator=g, device="cuda") * 0.1)
            want = [step() for _, step in pair]
            for graph in graphs if turn % 2 else graphs[::-1]:
                graph.replay()
            torch.cuda.synchronize()
            for w_, o_ in zip(want, outs):
                for a, c in zip(w_, o_):
                    assert torch.equal(a, c), (path, turn)
            pair[0][1]()
            torch.cuda.synchronize()
