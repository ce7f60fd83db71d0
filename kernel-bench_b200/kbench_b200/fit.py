"""Fit of the rates theta by Adam on the solver's implicit gradients, with what the fitted model says
about the families' origins.

    python -m kbench_b200.fit --config 1 --steps 50 --lr 0.05 --max-norm 1.0

A step is a forward solve, the root rows' scores, the backward solve and one clipped update.  Where the
species a family originated in is known (``observed``), minus ``weight`` times its log2 probability under
the root row is added to the loss, and its gradient goes into the backward solve as the root rows'
cotangent.  The reference fits theta with torch optimisers on the same gradients
(``newton/`` of the reference project); here a step makes no host synchronisation.
"""

from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from . import fitting, runtime, scoring


class FitResult(NamedTuple):
    theta: torch.Tensor             # [S, 3]
    objective: torch.Tensor         # [steps] before each update
    grad_norm: torch.Tensor         # [steps] of theta's gradient, before clipping
    scores: scoring.RowScores       # of the root rows at the last step's theta, before its update


def fit_rates(static, theta, col_weights, *, steps: int, lr: float = 0.05, max_norm: float = 1.0,
              weight_decay: float = 0.0, observed: Optional[torch.Tensor] = None, weight: float = 1.0,
              top: int = 3) -> FitResult:
    """``steps`` updates of a copy of ``theta``.  ``observed`` int64 [n_roots]: known origin columns (one
    outside [0, S): not known)."""
    if steps < 1:
        raise ValueError(f"steps must be at least 1 (got {steps})")
    theta = theta.detach().clone(memory_format=torch.contiguous_format)
    opt = fitting.Adam([theta], lr=lr, max_norm=max_norm, weight_decay=weight_decay)
    objective, norms = [], []
    for _ in range(steps):
        loss, saved = runtime.run_forward(static, theta, col_weights, check_errors=False)
        rows = saved["root_rows"]
        scores = scoring.score_rows(rows, observed, top=top)
        cotangent = None
        if observed is not None:
            loss = loss - weight * scores.given_log_prob.sum()
            cotangent = scoring.score_rows_backward(
                rows, scores.stats, None, observed, grad_given=torch.full_like(scores.given_log_prob, -weight))
        grad_theta, _ = runtime.run_backward(static, theta, col_weights, saved, check_errors=False,
                                             root_cotangent=cotangent)
        norms.append(opt.step([grad_theta]))
        objective.append(loss.reshape(()))
    runtime.check_errors(static)
    return FitResult(theta, torch.stack(objective), torch.stack(norms), scores)


def main():
    import argparse
    import json

    from . import gen
    ap = argparse.ArgumentParser()
    ap.add_argument("--config", type=int, default=1)
    ap.add_argument("--steps", type=int, default=50)
    ap.add_argument("--lr", type=float, default=0.05)
    ap.add_argument("--max-norm", type=float, default=1.0)
    ap.add_argument("--origin", type=int, default=None, help="known origin column of every family")
    ap.add_argument("--top", type=int, default=3)
    a = ap.parse_args()
    dev = torch.device("cuda:0")
    cap = gen.generate(a.config)
    static = runtime.make_static(cap, dev)
    theta, cw = cap["inputs"]["theta"].to(dev), cap["inputs"]["col_weights"].to(dev)
    roots = static.wave_layout["root_row_ids"]
    observed = None if a.origin is None else torch.full_like(roots, a.origin, dtype=torch.int64)
    r = fit_rates(static, theta, cw, steps=a.steps, lr=a.lr, max_norm=a.max_norm, observed=observed, top=a.top)
    s = r.scores
    columns, probs = ([[]] * len(s.entropy) if t is None else t.tolist() for t in (s.top_column, s.top_log_prob))
    print(json.dumps({
        "objective_first": float(r.objective[0]), "objective_last": float(r.objective[-1]),
        "grad_norm_last": float(r.grad_norm[-1]),
        "origins": [{"column": c, "log2_prob": [round(v, 4) for v in p], "entropy_bits": round(h, 4)} for c, p, h in
                    list(zip(columns, probs, s.entropy.tolist()))[:8]]}))


if __name__ == "__main__":
    main()
