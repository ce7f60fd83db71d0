"""The fit of theta (``kbench_b200.fit``) and the root rows' cotangent of the backward solve."""

import json
import math
import sys

import pytest
import torch

from kbench_b200 import fit, fitting, gen, runtime, scoring, tangent

pytestmark = pytest.mark.gpu


def _problem(cuda, engine="fused", pi_iters=32, neumann_terms=32):
    cap = gen.generate(gen.ProblemConfig("fit", 24, 30, 6, 40, 120, n_families=3), seed=5,
                       solver_options={"pi_iters": pi_iters, "neumann_terms": neumann_terms,
                                       "use_adjoint_pruning": False, "adjoint_pruning_threshold": 0.0})
    static = runtime.make_static(cap, cuda, engine=engine)
    return static, cap["inputs"]["theta"].to(cuda), cap["inputs"]["col_weights"].to(cuda)


def _supervised(static, theta, cw, observed, w):
    loss, saved = runtime.run_forward(static, theta, cw)
    s = scoring.score_rows(saved["root_rows"], observed)
    cot = scoring.score_rows_backward(saved["root_rows"], s.stats, s.entropy, observed,
                                      grad_given=torch.full_like(s.given_log_prob, -w),
                                      grad_entropy=torch.full_like(s.entropy, 0.3))
    return loss, saved, s, cot


@pytest.mark.parametrize("engine", ["fused", "wrappers"])
def test_root_cotangent_is_the_transposed_tangent(engine, cuda):
    """<V, grad with the cotangent - grad without> = <cotangent, root tangent along V>: the two are
    computed by the adjoint and the tangent solvers; they agree to the benchmark's acceptance of
    a tangent (rel 1e-3, here of the sum of the terms' sizes)."""
    static, theta, cw = _problem(cuda, engine)
    observed = torch.tensor([3, 0, 17], device=cuda)
    _, saved, _, cot = _supervised(static, theta, cw, observed, 2.0)
    base, _ = runtime.run_backward(static, theta, cw, saved)
    both, _ = runtime.run_backward(static, theta, cw, saved, root_cotangent=cot)
    fused, ft, fc = _problem(cuda)
    _, fsaved = runtime.run_forward(fused, ft, fc)
    V = torch.randn((6, *theta.shape), generator=torch.Generator().manual_seed(1)).to(cuda)
    roots = tangent.jvp_batch(fused, ft, V, fsaved)
    for v, dr in zip(V, roots):
        want = (cot.double() * dr.double()).sum()
        terms = v.double() * (both - base).double()
        assert abs(float(terms.sum() - want)) <= 1e-3 * float(terms.abs().sum())


def test_no_cotangent_changes_nothing(cuda):
    static, theta, cw = _problem(cuda)
    loss, saved = runtime.run_forward(static, theta, cw)
    a = runtime.run_backward(static, theta, cw, saved)
    b = runtime.run_backward(static, theta, cw, saved, root_cotangent=torch.zeros_like(saved["root_rows"]))
    assert torch.allclose(a[0], b[0], rtol=1e-4, atol=1e-6) and torch.allclose(a[1], b[1], rtol=1e-4, atol=1e-6)


def test_the_losss_own_cotangent(cuda):
    """With the gradient of +log mass as the root rows' cotangent the loss's own root term cancels, and
    with that of -log mass it doubles: differences from the plain gradient are opposite."""
    static, theta, cw = _problem(cuda)
    _, saved = runtime.run_forward(static, theta, cw)
    s = scoring.score_rows(saved["root_rows"])
    one = torch.ones_like(s.log_mass)
    grads = [runtime.run_backward(static, theta, cw, saved, root_cotangent=c)[0].double() for c in (
        scoring.score_rows_backward(saved["root_rows"], s.stats, None, grad_log_mass=one),
        torch.zeros_like(saved["root_rows"]),
        scoring.score_rows_backward(saved["root_rows"], s.stats, None, grad_log_mass=-one))]
    up, down = grads[0] - grads[1], grads[2] - grads[1]
    assert float((up + down).norm()) <= 1e-3 * float(down.norm())


def test_scores_are_the_losss_terms(cuda):
    """The loss is minus the root rows' log mass plus what the extinction vector adds."""
    static, theta, cw = _problem(cuda)
    loss, saved = runtime.run_forward(static, theta, cw)
    S = saved["root_rows"].shape[1]
    s = scoring.score_rows(saved["root_rows"], top=S if S <= 32 else 32)
    norm = torch.log2((1 - torch.exp2(saved["E"]).mean(-1)).clamp_min(torch.finfo(torch.float32).tiny))
    want = (-(s.log_mass - torch.log2(torch.tensor(float(S), device=cuda)) - norm)).sum()
    assert abs(float(loss) - float(want)) <= 1e-5 * abs(float(loss))


def test_fit_lowers_the_objective(cuda):
    static, theta, cw = _problem(cuda, pi_iters=8, neumann_terms=8)
    before = theta.clone()
    plain = fit.fit_rates(static, theta, cw, steps=25, lr=0.05, max_norm=1.0)
    assert torch.equal(theta, before) and plain.theta.shape == theta.shape
    assert float(plain.objective[-1]) < float(plain.objective[0])
    # the origin that the plain fit thinks least likely, made known
    observed = saved_worst = runtime.run_forward(static, plain.theta, cw)[1]["root_rows"].argmin(1)
    told = fit.fit_rates(static, theta, cw, steps=25, lr=0.05, max_norm=1.0, observed=observed, weight=5.0)
    assert float(told.objective[-1]) < float(told.objective[0])
    rows = runtime.run_forward(static, told.theta, cw)[1]["root_rows"]
    plain_lp = scoring.score_rows(runtime.run_forward(static, plain.theta, cw)[1]["root_rows"], saved_worst)
    assert float(scoring.score_rows(rows, observed).given_log_prob.sum()) > float(plain_lp.given_log_prob.sum())


def test_refusals(cuda):
    static, theta, cw = _problem(cuda)
    _, saved = runtime.run_forward(static, theta, cw)
    z = torch.zeros_like(saved["root_rows"])
    with pytest.raises(ValueError):
        runtime.run_backward(static, theta, cw, saved, root_cotangent=z[:, 1:])
    with pytest.raises(RuntimeError):
        runtime.run_backward(static, theta, cw, saved, root_cotangent=z.double())
    with pytest.raises(RuntimeError):
        runtime.run_backward(static, theta, cw, saved, root_cotangent=z.cpu())
    with pytest.raises(ValueError):
        fit.fit_rates(static, theta, cw, steps=0)


def test_command(cuda, capsys, monkeypatch):
    monkeypatch.setattr(sys, "argv", ["fit", "--config", "1", "--steps", "5", "--origin", "4"])
    fit.main()
    got = json.loads(capsys.readouterr().out)
    assert got["objective_last"] < got["objective_first"] and len(got["origins"][0]["column"]) == 3


def test_both_parameters_are_fitted(cuda):
    """Uniform column weights that an update makes different: the next solves take them as they are."""
    static, theta, cw = _problem(cuda, pi_iters=8, neumann_terms=8)
    assert bool((cw == cw[0]).all())
    opt = fitting.Adam([theta, cw], lr=0.05, max_norm=1.0)
    for _ in range(2):
        loss, saved = runtime.run_forward(static, theta, cw)
        grads = runtime.run_backward(static, theta, cw, saved)
        fresh = cw.clone()
        want, wsaved = runtime.run_forward(static, theta, fresh)
        wgrads = runtime.run_backward(static, theta, fresh, wsaved)
        # the same solves, up to the order of fp32 additions
        assert torch.allclose(loss, want, rtol=1e-6)
        assert torch.allclose(saved["root_rows"], wsaved["root_rows"], rtol=1e-5, atol=1e-5)
        for a, b in zip(grads, wgrads):
            assert torch.allclose(a, b, rtol=1e-4, atol=1e-6)
        runtime.run_forward(static, theta, cw)  # remembered once more for the tensor that is fitted
        opt.step(grads)
    assert not bool((cw == cw[0]).all())


def test_command_without_alternatives(cuda, capsys, monkeypatch):
    monkeypatch.setattr(sys, "argv", ["fit", "--config", "1", "--steps", "2", "--top", "0"])
    fit.main()
    got = json.loads(capsys.readouterr().out)
    assert got["origins"] and all(o["column"] == [] and o["log2_prob"] == [] and o["entropy_bits"] >= 0
                                  for o in got["origins"])


@pytest.mark.parametrize("engine", ["fused", "wrappers"])
def test_the_losss_own_cotangent_by_value(engine, cuda):
    """The cotangents of +- log mass change the gradient by +- that of the root rows' log mass, which the
    tangent solver gives along any direction (to the acceptance of a tangent, as above); with + the seed
    is zero and only the extinction vector's term is left, with - the root part doubles."""
    static, theta, cw = _problem(cuda, engine)
    _, saved = runtime.run_forward(static, theta, cw)
    rows = saved["root_rows"]
    s = scoring.score_rows(rows)
    cot = scoring.score_rows_backward(rows, s.stats, None, grad_log_mass=torch.ones_like(s.log_mass))
    base = runtime.run_backward(static, theta, cw, saved)[0].double()
    up, down = (runtime.run_backward(static, theta, cw, saved, root_cotangent=sign * cot)[0].double() - base
                for sign in (1.0, -1.0))
    fused, ft, fc = _problem(cuda)
    _, fsaved = runtime.run_forward(fused, ft, fc)
    V = torch.randn((6, *theta.shape), generator=torch.Generator().manual_seed(2)).to(cuda)
    V[0] = theta.sign() + 2.0  # all entries of one sign: the terms add up
    V[1] = 1.0
    wants = []
    for v, dr in zip(V, tangent.jvp_batch(fused, ft, V, fsaved)):
        want = float((torch.softmax(fsaved["root_rows"].double() * math.log(2.0), 1) * dr.double()).sum())
        for sign, change in ((1.0, up), (-1.0, down)):
            terms = v.double() * change
            assert abs(sign * float(terms.sum()) - want) <= 1e-3 * float(terms.abs().sum())
        wants.append(abs(want))
    assert min(wants) > 0.0
    # a zero seed: what is left does not depend on the root rows at all
    zero = runtime.run_backward(static, theta, cw, saved, root_cotangent=cot)[0].double()
    twice = runtime.run_backward(static, theta, cw, saved, root_cotangent=cot * 2.0)[0].double()
    assert float((twice - zero - up).norm()) <= 1e-3 * float(up.norm())
