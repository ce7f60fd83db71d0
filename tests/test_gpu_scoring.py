"""Row scores (``kbench_b200.scoring``) and their gradient against a plain evaluation in 64 bits.

Tolerances, with e = 2^-24 (half an ulp of fp32):
* the sum Sigma adds terms 2^z with z = (x - m) scale: each carries e |z| ln 2 per rounding of z (at most
  three) and 4 e of the exponential; the weighted mean of |z| is at most log2 S (the entropy is not
  negative).  The additions of positive terms add at most e per addition of the longest chain, 96.
  Relative error of Sigma: REL(S) = e (3 log2 S + 100).
* a log probability (x - m) - log Sigma: REL / ln 2 bits and the roundings of its two terms;
* the entropy log2 Sigma - (sum w z) / Sigma: REL / ln 2 and 2 REL of a mean of at most log2 S;
* the gradient p (a - G - h ln 2 (z + bits)) + g: p to e (3 |z| + 16), the bracket by its terms' sizes,
  then the rounding to the rows' dtype.
"""

import math

import pytest
import torch

from kbench_b200 import scoring

pytestmark = pytest.mark.gpu

EPS = 2.0 ** -24
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
HALF_ULP = {t: torch.finfo(t).eps / 2 for t in DTYPES.values()}
SMALLEST = {torch.float32: 2.0 ** -126, torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -25}
SHAPES = [(1, 1), (1, 2), (3, 31), (2, 63), (5, 79), (7, 255), (4, 511), (3, 1023), (2, 4095), (3, 8192), (2, 33333),
          (1, 131071), (300, 17), (1200, 129), (2500, 63)]


def rel(S):
    return EPS * (3.0 * math.log2(S + 1) + 100.0)


def make_rows(R, S, kind, dtype, device, seed=0):
    g = torch.Generator(device="cpu").manual_seed(1000 * seed + 17 * R + S)
    x = torch.randn((R, S), generator=g) * 3.0
    if kind == "solver":
        x += torch.rand((R, 1), generator=g) * -300.0 - 5.0
    elif kind == "masked":
        x[torch.rand((R, S), generator=g) < 0.4] = -math.inf
        x[::3] = -math.inf
    elif kind == "one":  # a single possible column
        keep = torch.randint(0, max(S, 1), (R, 1), generator=g)
        x = torch.full((R, S), -math.inf).scatter(1, keep, x[:, :1])
    elif kind == "lowest":  # masks of the type's lowest value, some rows wholly so
        low = torch.finfo(dtype).min
        x[torch.rand((R, S), generator=g) < 0.4] = low
        x[::2] = low
    elif kind == "ties":
        x = torch.round(x) * 0.5
        x[torch.rand((R, S), generator=g) < 0.3] = -0.0
    elif kind == "equal":
        x[:] = -7.25
    elif kind == "ascending":
        x = torch.sort(x, dim=1).values
    elif kind == "descending":
        x = torch.sort(x, dim=1, descending=True).values
    else:
        assert kind == "plain"
    return x.to(dtype).to(device)


def reference(x, given, top, base):
    """The scores in 64 bits, unit of the base."""
    x = x.double()
    R, S = x.shape
    u = math.log(2.0) if base == 2 else 1.0
    m = x.amax(1) if S else torch.full((R,), -math.inf, dtype=x.dtype, device=x.device)
    empty = torch.isneginf(m)
    ms = torch.where(empty, torch.zeros_like(m), m)
    w = torch.exp((x - ms[:, None]) * u)
    total = w.sum(1)
    lp = torch.where(empty[:, None], torch.full_like(x, -math.inf), (x - ms[:, None]) - (total.log() / u)[:, None])
    p = torch.where(empty[:, None], torch.zeros_like(w), w / total[:, None])
    entropy = torch.special.entr(p).sum(1) / u
    out = {"log_mass": torch.where(empty, m, ms + total.log() / u), "entropy": entropy,
           "m": m, "total": total, "lp": lp, "p": p, "u": u}
    if given is not None:
        at = given.long().reshape(R, -1)
        inside = (at >= 0) & (at < S)
        got = torch.zeros(at.shape, dtype=x.dtype, device=x.device)
        if S:
            got = torch.where(inside, lp.gather(1, at.clamp(0, S - 1)), got)
        out["given"] = got.reshape(given.shape)
    if top:
        k = min(top, S)
        order = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :k]
        out["column"] = torch.cat([order, torch.full((R, top - k), -1, dtype=order.dtype, device=x.device)], 1)
        out["top"] = torch.cat([lp.gather(1, order), torch.full((R, top - k), -math.inf, dtype=x.dtype,
                                                               device=x.device)], 1)
    return out


def near(name, got, ref, tol):
    got, ref = got.double(), ref.double()
    tol = torch.as_tensor(tol, dtype=torch.float64, device=ref.device).expand_as(ref)
    assert got.shape == ref.shape, name
    special = ~torch.isfinite(ref)
    assert torch.equal(torch.isnan(got), torch.isnan(ref)), f"{name}: NaN pattern"
    keep = special & ~torch.isnan(ref)
    assert torch.equal(got[keep], ref[keep]), f"{name}: infinities"
    d = (got - ref).abs()[~special]
    worst = (d / tol[~special].clamp_min(1e-300)).max() if d.numel() else torch.tensor(0.0)
    assert bool((d <= tol[~special]).all()), f"{name}: worst error {float(worst):.3g} of its tolerance"


def check_scores(s, x, given, top, base):
    ref = reference(x, given, top, base)
    S = x.shape[1]
    unit = 1.0 if base == 2 else math.log(2.0)
    r, logs = rel(S), math.log2(S + 2)
    lp_tol = lambda lp: unit * r / math.log(2.0) + 4 * EPS * (torch.nan_to_num(lp.abs(), posinf=0.0) + 2 * logs * unit + 1)
    near("stats max", s.stats[:, 0], ref["m"], 0.0)
    near("stats sum", s.stats[:, 1], ref["total"], r * ref["total"])
    near("log_mass", s.log_mass, ref["log_mass"],
         unit * r / math.log(2.0) + 2 * EPS * torch.nan_to_num(ref["log_mass"].abs(), posinf=0.0) + 2 * EPS * logs)
    near("entropy", s.entropy, ref["entropy"], unit * (r / math.log(2.0) + 2 * r * logs + 4 * EPS * logs))
    if given is not None:
        near("given", s.given_log_prob, ref["given"], lp_tol(ref["given"]))
    else:
        assert s.given_log_prob is None
    if top:
        assert torch.equal(s.top_column, ref["column"])
        near("top", s.top_log_prob, ref["top"], lp_tol(ref["top"]))
    else:
        assert s.top_log_prob is None and s.top_column is None


def make_given(R, S, T, device, seed=0):
    g = torch.Generator(device="cpu").manual_seed(seed + 5)
    return torch.randint(-2, S + 2, (R, T), generator=g).to(device)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("base", [2, "e"])
def test_scores(shape, dtype, base, cuda):
    R, S = shape
    x = make_rows(R, S, "solver" if base == 2 else "plain", DTYPES[dtype], cuda)
    given = make_given(R, S, 3, cuda)
    check_scores(scoring.score_rows(x, given, top=8, base=base), x, given, 8, base)


@pytest.mark.parametrize("kind", ["masked", "one", "lowest", "ties", "equal", "ascending", "descending"])
@pytest.mark.parametrize("shape", [(1, 1), (9, 33), (4, 700), (2, 4095), (3, 40000), (1300, 600)])
@pytest.mark.parametrize("dtype", list(DTYPES))
def test_hard_rows(kind, shape, dtype, cuda):
    R, S = shape
    x = make_rows(R, S, kind, DTYPES[dtype], cuda)
    given = make_given(R, S, 2, cuda)
    for top in (1, 5, 32):
        check_scores(scoring.score_rows(x, given, top=top), x, given, top, 2)


@pytest.mark.parametrize("top", [0, 1, 2, 7, 16, 20, 31, 32])
@pytest.mark.parametrize("shape", [(3, 5), (2, 200), (2, 3000), (1, 70001), (700, 300)])
def test_tops_and_no_given(top, shape, cuda):
    x = make_rows(*shape, "solver", torch.float32, cuda, seed=top)
    check_scores(scoring.score_rows(x, top=top), x, None, top, 2)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("rows", [1, 3])
def test_very_long_rows(rows, dtype, cuda):
    """Five million columns: 153 batches a warp, so 200 additions in the longest chain instead of 96;
    the offset of the rows (300 bits) leaves 16-bit rows a handful of values, equal over long stretches."""
    S = 5000011
    x = make_rows(rows, S, "solver", DTYPES[dtype], cuda)
    x[-1, S // 3:S // 2] = -math.inf
    given = make_given(rows, S, 4, cuda)
    given[:, 0] = S - 1
    s = scoring.score_rows(x, given, top=32)
    ref = reference(x, given, 32, 2)
    r = EPS * (3.0 * math.log2(S) + 200.0)
    assert torch.equal(s.top_column, ref["column"])
    near("stats max", s.stats[:, 0], ref["m"], 0.0)
    near("stats sum", s.stats[:, 1], ref["total"], r * ref["total"])
    near("entropy", s.entropy, ref["entropy"], r / math.log(2.0) + 2 * r * 24 + 4 * EPS * 24)
    near("given", s.given_log_prob, ref["given"], r / math.log(2.0) + 4 * EPS * (torch.nan_to_num(ref["given"].abs(), posinf=0.0) + 50))
    g = torch.ones_like(s.given_log_prob)
    got = scoring.score_rows_backward(x, s.stats, s.entropy, given, grad_given=g).double()
    inside = (given >= 0) & (given < S)
    at = given.clamp(0, S - 1)
    live = (inside & ~torch.isneginf(x.gather(1, at))).double()
    want = torch.zeros_like(ref["p"]).scatter_add_(1, at, live) - ref["p"] * live.sum(1, keepdim=True)
    tol = ref["p"] * 4 * (2 * r + 60 * EPS) + 8 * EPS * want.abs() + HALF_ULP[x.dtype] * want.abs() * 1.01 + SMALLEST[x.dtype]
    near("grad", got, want, tol)


def test_tops_in_adverse_places(cuda):
    """The largest entries together in one stretch, at either end, or one to every 128 columns."""
    S = 50000
    x = make_rows(6, S, "plain", torch.float32, cuda)
    ramp = torch.arange(64, device=cuda, dtype=torch.float32) + 50.0
    x[0, :64] = ramp
    x[1, -64:] = ramp
    x[2, 25000:25064] = ramp.flip(0)
    x[3, 3:3 + 64 * 128:128] = ramp
    x[4, 1::512] = torch.arange(len(range(1, S, 512)), device=cuda, dtype=torch.float32) + 50.0
    x[5, ::2] = 60.0
    for top in (4, 20, 32):
        check_scores(scoring.score_rows(x, top=top), x, None, top, 2)


@pytest.mark.parametrize("T", [1, 2, 17, 32])
@pytest.mark.parametrize("index", [torch.int64, torch.int32])
def test_given_forms(T, index, cuda):
    x = make_rows(6, 321, "masked", torch.float32, cuda)
    given = make_given(6, 321, T, cuda).to(index)
    check_scores(scoring.score_rows(x, given), x, given, 0, 2)
    one = given[:, 0]
    s = scoring.score_rows(x, one)
    assert s.given_log_prob.shape == (6,)
    check_scores(s, x, one, 0, 2)


def strided(kind, R, S, dtype, device):
    x = make_rows(R, S, "solver", dtype, device)
    if kind == "padded":
        buf = torch.full((R, S + 13), float("nan"), dtype=dtype, device=device)
        v = buf[:, 5:5 + S]
    elif kind == "shifted":  # starts one entry into an allocation
        v = torch.full((R * S + 1,), float("nan"), dtype=dtype, device=device)[1:].view(R, S)
    elif kind == "transposed":
        v = torch.empty((S, R), dtype=dtype, device=device).t()
    else:  # one row repeated
        return x[:1].expand(R, S)
    v.copy_(x)
    return v


@pytest.mark.parametrize("kind", ["padded", "shifted", "transposed", "expanded"])
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("shape", [(3, 67), (2, 4099), (1400, 130)])
def test_strides(kind, dtype, shape, cuda):
    x = strided(kind, *shape, DTYPES[dtype], cuda)
    given = make_given(*shape, 2, cuda)
    s = scoring.score_rows(x, given, top=6)
    check_scores(s, x, given, 6, 2)
    check_grad(x, given, 2, s)


def test_empty_shapes(cuda):
    s = scoring.score_rows(torch.empty((0, 7), device=cuda), top=3)
    assert s.log_mass.shape == (0,) and s.top_column.shape == (0, 3)
    x = torch.empty((3, 0), device=cuda)
    given = torch.zeros(3, dtype=torch.int64, device=cuda)
    s = scoring.score_rows(x, given, top=2)
    check_scores(s, x, given, 2, 2)
    assert scoring.score_rows_backward(x, s.stats, s.entropy).shape == (3, 0)


@pytest.mark.parametrize("bad", [math.nan, -math.nan, math.inf])
@pytest.mark.parametrize("S", [1, 40, 5000, 100000])
def test_rows_that_are_no_distribution(bad, S, cuda):
    x = make_rows(3, S, "plain", torch.float32, cuda)
    clean = x.clone()
    x[1, S // 2] = bad
    given = torch.zeros((3, 1), dtype=torch.int64, device=cuda)
    s = scoring.score_rows(x, given, top=4)
    for t in (s.log_mass, s.entropy, s.given_log_prob, s.top_log_prob, s.stats):
        assert bool(torch.isnan(t[1]).all())
    assert bool((s.top_column[1] == -1).all())
    want = scoring.score_rows(clean, given, top=4)
    for t, w in zip(s, want):  # the neighbours are untouched
        assert torch.equal(t[0], w[0]) and torch.equal(t[2], w[2])
    g = scoring.score_rows_backward(x, s.stats, s.entropy, grad_log_mass=torch.ones(3, device=cuda))
    assert bool(torch.isnan(g[1]).all()) and bool(torch.isfinite(g[0]).all())


# ---- the gradient ------------------------------------------------------------------------------

def objective(x, given, a, g, h, base):
    """sum a log_mass + sum g log p(given) + sum h entropy in 64 bits (rows with a possible column)."""
    ref = reference(x, given, 0, base)
    some = ~torch.isneginf(ref["m"])
    lp = ref["given"].reshape(x.shape[0], -1)
    lp = torch.where(torch.isneginf(lp), torch.zeros_like(lp), lp)
    return (a.double()[some] * ref["log_mass"][some]).sum() + (g.double() * lp)[some].sum() + \
        (h.double() * ref["entropy"])[some].sum()


def cotangents(R, T, device, seed=3):
    c = torch.Generator(device="cpu").manual_seed(seed)
    return (torch.randn(R, generator=c).to(device), torch.randn((R, T), generator=c).to(device),
            torch.randn(R, generator=c).to(device))


def check_grad(x, given, base, s, out=None, which=(True, True, True)):
    R, S = x.shape
    a, g, h = cotangents(R, given.shape[1], x.device)
    got = scoring.score_rows_backward(
        x, s.stats, s.entropy, given, grad_log_mass=a if which[0] else None, grad_given=g if which[1] else None,
        grad_entropy=h if which[2] else None, base=base, out=out)
    a, g, h = (t * float(w) for t, w in zip((a, g, h), which))
    ref = reference(x, given, 0, base)
    p, lp, u = ref["p"], ref["lp"], ref["u"]
    at = given.long().clamp(0, S - 1)
    live = (given >= 0) & (given < S) & ~torch.isneginf(x.gather(1, at))
    gl = torch.where(live, g, torch.zeros_like(g)).double()
    hot = torch.zeros_like(p).scatter_add_(1, at, gl)
    size = torch.zeros_like(p).scatter_add_(1, at, gl.abs())
    nats = torch.where(p > 0, lp * u, torch.zeros_like(lp))
    H = ref["entropy"][:, None] * u
    want = hot + p * (a.double()[:, None] - gl.sum(1, keepdim=True) - h.double()[:, None] * (nats + H))
    logs = math.log(S + 2)
    scale = a.double().abs()[:, None] + gl.abs().sum(1, keepdim=True) + h.double().abs()[:, None] * (nats.abs() + H + logs)
    # the stats and the entropy carry the forward's own errors
    tol = p * scale * (EPS * (3 * nats.abs() / math.log(2) + 16) + 2 * rel(S) * (1 + logs)) + 8 * EPS * size
    tol = tol + HALF_ULP[x.dtype] * (want.abs() + tol) + SMALLEST[x.dtype]
    assert got.dtype == x.dtype and got.shape == x.shape
    near("grad", got, want, tol)
    assert bool((got[torch.isneginf(x)] == 0).all())
    return got


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("base", [2, "e"])
def test_gradient(shape, dtype, base, cuda):
    R, S = shape
    x = make_rows(R, S, "solver" if base == 2 else "plain", DTYPES[dtype], cuda)
    given = make_given(R, S, 3, cuda)
    check_grad(x, given, base, scoring.score_rows(x, given, base=base))


@pytest.mark.parametrize("kind", ["masked", "one", "lowest", "equal"])
@pytest.mark.parametrize("shape", [(1, 1), (9, 33), (4, 700), (2, 4095), (1300, 600)])
def test_gradient_hard_rows(kind, shape, cuda):
    x = make_rows(*shape, kind, torch.float32, cuda)
    given = make_given(*shape, 4, cuda)
    given[:, 1] = given[:, 0]  # the same column twice
    check_grad(x, given, 2, scoring.score_rows(x, given))


@pytest.mark.parametrize("which", [(True, False, False), (False, True, False), (False, False, True),
                                   (False, False, False)])
@pytest.mark.parametrize("T", [1, 32])
def test_gradient_parts(which, T, cuda):
    x = make_rows(5, 900, "solver", torch.float32, cuda)
    given = make_given(5, 900, T, cuda)
    check_grad(x, given, 2, scoring.score_rows(x, given), which=which)


@pytest.mark.parametrize("dtype", list(DTYPES))
def test_gradient_into_other_strides(dtype, cuda):
    """An output whose rows start at other distances from a 16-byte boundary than the input's."""
    x = make_rows(5, 1025, "solver", DTYPES[dtype], cuda)
    given = make_given(5, 1025, 2, cuda)
    buf = torch.full((5, 1040), 7.0, dtype=x.dtype, device=cuda)
    check_grad(x, given, 2, scoring.score_rows(x, given), out=buf[:, 3:1028])
    assert bool((buf[:, :3] == 7).all()) and bool((buf[:, 1028:] == 7).all())


@pytest.mark.parametrize("base", [2, "e"])
@pytest.mark.parametrize("shape", [(1, 63), (3, 1023)])
def test_gradient_by_differences(base, shape, cuda):
    """Central differences of the 64-bit objective along random directions: their own error is
    O(step^2) of third derivatives (1e-10 here) and 1e-16 / step of the objective's size."""
    R, S = shape
    x = make_rows(R, S, "plain", torch.float32, cuda)
    given = make_given(R, S, 2, cuda)
    a, g, h = cotangents(R, 2, cuda)
    s = scoring.score_rows(x, given, base=base)
    grad = scoring.score_rows_backward(x, s.stats, s.entropy, given, grad_log_mass=a, grad_given=g, grad_entropy=h,
                                       base=base).double()
    gen = torch.Generator(device="cpu").manual_seed(8)
    for _ in range(4):
        d = torch.randn((R, S), generator=gen, dtype=torch.float64).to(cuda)
        step = 1e-5
        up, down = (objective(x.double() + t * step * d, given, a, g, h, base) for t in (1, -1))
        want = float(up - down) / (2 * step)
        size = float((grad * d).abs().sum())
        assert abs(float((grad * d).sum()) - want) <= 1e-5 * size + 1e-7


def test_loss_cotangent_is_the_solvers(cuda):
    """The solver's own root cotangent is the gradient of minus the log mass."""
    from kbench_b200 import glue
    x = make_rows(7, 1023, "solver", torch.float32, cuda)
    s = scoring.score_rows(x)
    got = scoring.score_rows_backward(x, s.stats, None, grad_log_mass=torch.full((7,), -1.0, device=cuda))
    # the solver forms 2^(x - log mass) from the rounded log mass (about 300): 2^-24 * 300 * ln 2 relative
    assert torch.allclose(got, glue.root_rhs(x, torch.arange(7, device=cuda)), rtol=4e-5, atol=1e-30)


# ---- use ---------------------------------------------------------------------------------------

def test_offsets_past_32_bits(cuda):
    R, S = 70000, 32771  # 2.29e9 entries
    x = torch.full((R, S), -3.0, dtype=torch.bfloat16, device=cuda)
    tail = make_rows(5, S, "plain", torch.bfloat16, cuda)
    x[-5:] = tail
    given = torch.full((R,), 11, dtype=torch.int64, device=cuda)
    s = scoring.score_rows(x, given, top=4)
    check_scores(scoring.RowScores(*(t[-5:] for t in s)), tail, given[-5:], 4, 2)
    out = scoring.score_rows_backward(x, s.stats, s.entropy, given, grad_given=torch.ones(R, device=cuda))
    del x
    want = scoring.score_rows_backward(tail, s.stats[-5:], s.entropy[-5:], given[-5:],
                                       grad_given=torch.ones(5, device=cuda))
    assert torch.equal(out[-5:], want)


def test_runs_repeat_bitwise_and_on_other_streams(cuda):
    for shape in ((2000, 700), (3, 100000)):
        x = make_rows(*shape, "solver", torch.float32, cuda)
        given = make_given(*shape, 3, cuda)
        one = scoring.score_rows(x, given, top=9)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            two = scoring.score_rows(x, given, top=9)
            grad = scoring.score_rows_backward(x, two.stats, two.entropy, given, grad_entropy=two.log_mass)
        torch.cuda.current_stream().wait_stream(side)
        for a, b in zip(one, two):
            assert torch.equal(a, b)
        assert torch.equal(grad, scoring.score_rows_backward(x, one.stats, one.entropy, given,
                                                             grad_entropy=one.log_mass))


def test_graph_capture(cuda):
    x = make_rows(40, 1023, "solver", torch.float32, cuda)
    given = make_given(40, 1023, 1, cuda)
    scoring.score_rows(x, given, top=3)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        s = scoring.score_rows(x, given, top=3)
    x.copy_(make_rows(40, 1023, "solver", torch.float32, cuda, seed=9))
    graph.replay()
    check_scores(s, x, given, 3, 2)


def test_refusals(cuda):
    x = torch.zeros((4, 9), device=cuda)
    given = torch.zeros(4, dtype=torch.int64, device=cuda)
    s = scoring.score_rows(x, given)
    for exc, call in (
        (RuntimeError, lambda: scoring.score_rows(x.cpu())),
        (RuntimeError, lambda: scoring.score_rows(x.double())),
        (ValueError, lambda: scoring.score_rows(x[0])),
        (ValueError, lambda: scoring.score_rows(x, top=33)),
        (ValueError, lambda: scoring.score_rows(x, top=-1)),
        (ValueError, lambda: scoring.score_rows(x, base=10)),
        (ValueError, lambda: scoring.score_rows(x, given[:3])),
        (ValueError, lambda: scoring.score_rows(x, given.float())),
        (RuntimeError, lambda: scoring.score_rows(x, given.cpu())),
        (ValueError, lambda: scoring.score_rows(x, given[:, None].expand(4, 33))),
        (ValueError, lambda: scoring.score_rows_backward(x, None, s.entropy)),
        (ValueError, lambda: scoring.score_rows_backward(x, s.stats[:3], s.entropy)),
        (RuntimeError, lambda: scoring.score_rows_backward(x, s.stats.double(), s.entropy)),
        (ValueError, lambda: scoring.score_rows_backward(x, s.stats, None, grad_entropy=s.entropy)),
        (ValueError, lambda: scoring.score_rows_backward(x, s.stats, s.entropy, grad_given=s.entropy)),
        (ValueError, lambda: scoring.score_rows_backward(x, s.stats, s.entropy, given, grad_given=s.stats)),
        (ValueError, lambda: scoring.score_rows_backward(x, s.stats, s.entropy, out=x)),
        (ValueError, lambda: scoring.score_rows_backward(x, s.stats, s.entropy, out=x.new_empty(9, 4).t())),
        (ValueError, lambda: scoring.score_rows_backward(x, s.stats, s.entropy, out=x.new_empty(1, 9).expand(4, 9))),
        (RuntimeError, lambda: scoring.score_rows_backward(x, s.stats, s.entropy, out=x.bfloat16())),
    ):
        with pytest.raises(exc):
            call()


@pytest.mark.parametrize("strided", [False, True])
def test_gradient_buffer_gets_a_new_version(strided, cuda):
    x = make_rows(5, 300, "solver", torch.float32, cuda)
    rows = x.t().contiguous().t() if strided else x
    s = scoring.score_rows(rows)
    out = torch.empty_like(x)
    before, kept = out._version, rows._version
    assert scoring.score_rows_backward(rows, s.stats, None, grad_log_mass=s.log_mass, out=out) is out
    assert out._version > before and rows._version == kept


def test_rows_past_the_longest_are_refused(cuda):
    x = torch.zeros((2, 1), dtype=torch.bfloat16, device=cuda)
    for S in ((1 << 30) + 1, 1 << 32):
        with pytest.raises(ValueError, match="columns"):
            scoring.score_rows(x.expand(2, S))
        with pytest.raises(ValueError, match="columns"):
            scoring.score_rows_backward(x.expand(2, S), torch.zeros((2, 2), device=cuda), None)


def test_outputs_that_do_not_fit_are_out_of_memory(cuda):
    """The allocator's own exception, with nothing launched: 205 GB of alternatives."""
    rows = torch.zeros((1, 4), device=cuda).expand(1_600_000_000, 4)
    with pytest.raises(torch.OutOfMemoryError):
        scoring.score_rows(rows, top=32)
    torch.cuda.empty_cache()


def test_tops_past_an_integer_are_refused(cuda):
    x = torch.zeros((4, 9), device=cuda)
    for top in (1 << 31, -(1 << 40)):
        with pytest.raises(ValueError):
            scoring.score_rows(x, top=top)


def test_output_on_the_rows_through_another_storage_is_refused(cuda):
    flat = torch.zeros(100, device=cuda)
    rows = flat[:60].view(6, 10)
    s = scoring.score_rows(rows)
    for at in (0, 30):
        out = torch.from_dlpack(flat[at:at + 60]).view(6, 10)
        with pytest.raises(ValueError):
            scoring.score_rows_backward(rows, s.stats, None, grad_log_mass=s.log_mass, out=out)
    assert not bool(flat.any())


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("S", [5, 63, 100, 250, 700, 4099])
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_impossible_columns_keep_zero_beside_any_cotangent(S, dtype, bad, cuda):
    """Rows of -inf alone have log mass -inf, whose functions have cotangents that are not finite."""
    x = make_rows(6, S, "plain", DTYPES[dtype], cuda)
    x[1], x[4] = -math.inf, -math.inf
    x[2, ::2], x[3, 1:] = -math.inf, -math.inf
    given = torch.zeros((6, 2), dtype=torch.int64, device=cuda)
    given[:, 1] = S // 2
    s = scoring.score_rows(x, given)
    one = torch.ones(6, device=cuda)
    cot = one.clone()
    cot[[1, 2, 4]] = bad
    for k in ("grad_log_mass", "grad_entropy", "grad_given"):
        got = scoring.score_rows_backward(x, s.stats, s.entropy, given, **{k: cot[:, None].repeat(1, 2) if k == "grad_given" else cot})
        assert bool((got[torch.isneginf(x)] == 0).all()), k
        want = scoring.score_rows_backward(x, s.stats, s.entropy, given, **{k: one[:, None].repeat(1, 2) if k == "grad_given" else one})
        for r in (0, 3, 5):
            assert torch.equal(got[r], want[r])
        # the possible columns of row 2 follow the formula: a cotangent at impossible given columns does not count
        live = got[2][~torch.isneginf(x[2])]
        counts = k != "grad_given" or bool((x[2, given[2]] > -math.inf).any())
        if live.numel() > 2:
            assert bool(torch.isfinite(live).all()) != counts


# ---- every form of the kernels -----------------------------------------------------------------

# rows past 1,024 columns: a warp a row with two batches under way (the first three) and one; four warps a row;
# eight, some of them without a batch in 16 bits; a CTA a row of many
FORMS = [(3, 1400), (1000, 4095), (2300, 5001), (2500, 4095), (500, 8191), (800, 5003), (400, 5003), (1000, 24001)]


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("shape", FORMS)
@pytest.mark.parametrize("kind,base", [("solver", 2), ("plain", "e"), ("masked", 2), ("masked", "e"), ("ties", 2), ("one", 2)])
def test_forms(shape, dtype, kind, base, cuda):
    x = make_rows(*shape, kind, DTYPES[dtype], cuda, seed=4)
    given = make_given(*shape, 2, cuda)
    ref = None
    for top in (0, 1, 8, 32):
        s = scoring.score_rows(x, given, top=top, base=base)
        if ref is None:
            check_scores(s, x, given, 0, base)
            wide = scoring.score_rows(x, given, top=32, base=base)
            check_scores(wide, x, given, 32, base)
            ref = wide
        else:  # the same row sums, and the head of the same list
            for a, b in zip((s.log_mass, s.entropy, s.given_log_prob, s.stats, s.top_log_prob, s.top_column),
                            (ref.log_mass, ref.entropy, ref.given_log_prob, ref.stats, ref.top_log_prob[:, :top],
                             ref.top_column[:, :top])):
                assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("shape", [(3, 1400), (5000, 257), (5000, 1023), (5000, 4095), (500, 8191), (2500, 9001)])
@pytest.mark.parametrize("kind,base", [("solver", 2), ("plain", "e"), ("masked", 2), ("masked", "e")])
def test_gradient_forms(shape, dtype, kind, base, cuda):
    x = make_rows(*shape, kind, DTYPES[dtype], cuda, seed=6)
    given = make_given(*shape, 3, cuda)
    given[:, 2] = given[:, 0]
    check_grad(x, given, base, scoring.score_rows(x, given, base=base))


@pytest.mark.parametrize("shape", [(40, 63), (40, 1023)])
def test_gradient_graph_capture(shape, cuda):
    x = make_rows(*shape, "solver", torch.float32, cuda)
    given = make_given(*shape, 2, cuda)
    a, g, h = cotangents(shape[0], 2, cuda)

    def step():
        s = scoring.score_rows(x, given)
        return scoring.score_rows_backward(x, s.stats, s.entropy, given, grad_log_mass=a, grad_given=g, grad_entropy=h)
    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    x.copy_(make_rows(*shape, "solver", torch.float32, cuda, seed=9))
    graph.replay()
    assert torch.equal(got, step())
