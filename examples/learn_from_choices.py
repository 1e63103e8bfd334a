"""Boosted trees that learn from choices, on one GPU.

    python examples/learn_from_choices.py [--rows 20000] [--rounds 30]

Three ways to train without a label per row, each a loop of "evaluate a loss on
the training margins, boost one round on its gradient":

  rank      scores from pairs of rows of which one was preferred
  episodes  a policy from pairs of action sequences of which one was preferred
  policy    a policy from sampled actions and their rewards, held near the one
            it started from
"""
from __future__ import annotations

import argparse
import math
import pathlib
import sys

import torch

sys.path.insert(0, str(pathlib.Path(__file__).resolve().parents[1] / "decision-programs_b200"))
import dp_gbdt as dp  # noqa: E402

ACTIONS = 4


def table(rows: int, seed: int):
    gen = torch.Generator("cuda").manual_seed(seed)
    return torch.randn(rows, 6, generator=gen, device="cuda"), gen


def best_action(x):
    """The action that pays in each row, known to the examples alone."""
    return (x[:, 0] > 0).int() * 2 + (x[:, 1] * x[:, 2] > 0).int()


def policy_model(d):
    return dp.Booster({"objective": "multi:softprob", "num_class": ACTIONS, "max_depth": 4, "eta": 0.5}, [d])


def sample(margin, gen):
    return torch.multinomial(torch.softmax(margin, 1), 1, generator=gen)[:, 0].int()


def rank(rows: int, rounds: int) -> tuple[float, float]:
    """Mean loss of the first and the last round."""
    x, gen = table(rows, 0)
    hidden = x[:, 0] + 0.5 * x[:, 1] * x[:, 2]
    a = torch.randint(0, rows, (8 * rows,), generator=gen, device="cuda")
    b = (a + torch.randint(1, rows, (8 * rows,), generator=gen, device="cuda")) % rows
    wins = hidden[a] > hidden[b]
    pairs = torch.stack([torch.where(wins, a, b), torch.where(wins, b, a)], 1).int()
    plan = dp.PreferencePairs(pairs, rows)  # checked and laid out once for all rounds
    d = dp.DMatrix.from_torch(x)            # no labels
    model = dp.Booster({"objective": "reg:squarederror", "max_depth": 5, "eta": 0.3, "base_score": 0}, [d])
    losses = []
    for i in range(rounds):
        r = plan.loss(model.train_margin(d)[:, 0], smoothing=0.01, hess=True)
        losses.append(r.loss.mean().item())
        model.boost(d, i, r.grad, r.hess)
    return losses[0], losses[-1]


def episodes(rows: int, rounds: int) -> tuple[float, float]:
    """Probability that the policy gives the paying action, before and after."""
    x, gen = table(rows, 1)
    d = dp.DMatrix.from_torch(x)
    model = policy_model(d)
    # episodes of one to twelve rows; of each two, the one that earned more a row is preferred
    cut = torch.randint(1, 13, (rows,), generator=gen, device="cuda").cumsum(0)
    begin = torch.cat([torch.zeros(1, dtype=torch.int64, device="cuda"), cut[cut <= rows]])
    begin = begin[: (begin.numel() - 1) // 2 * 2 + 1]
    start = model.train_margin(d)
    action = sample(start, gen)
    reward = torch.cat([torch.zeros(1, device="cuda"), (action == best_action(x)).float().cumsum(0)])
    earned = (reward[begin[1:]] - reward[begin[:-1]]) / begin.diff()
    sign = torch.sign(earned[0::2] - earned[1::2])
    swap = sign < 0
    ref, _ = dp.log_prob(start, action)
    inside = torch.arange(rows, device="cuda")
    pair = (torch.searchsorted(begin, inside, right=True) - 1).clamp(0, begin.numel() - 2) // 2
    turn = torch.where(swap[pair], -1.0, 1.0)  # the loss prefers the first of a pair: swapped pairs enter negated
    weight = sign.abs()                        # ties count for nothing
    before = torch.softmax(start, 1).gather(1, best_action(x).long()[:, None]).mean().item()
    for i in range(rounds):
        margin = model.train_margin(d)
        logp, norm = dp.log_prob(margin, action)
        r = dp.preference_loss(logp * turn, ref_score=ref * turn, item_begin=begin, weight=weight, beta=0.5)
        grad, hess = dp.log_prob_grad(margin, action, norm, r.grad * turn, hess=True)
        model.boost(d, i, grad, hess)
    after = torch.softmax(model.train_margin(d), 1).gather(1, best_action(x).long()[:, None]).mean().item()
    return before, after


def policy(rows: int, rounds: int) -> tuple[float, float]:
    """Mean reward of the actions sampled first and last."""
    x, gen = table(rows, 2)
    d = dp.DMatrix.from_torch(x)
    model = policy_model(d)
    start, rewards, step = model.train_margin(d), [], 0
    for _ in range(max(2, rounds // 3)):
        margin = model.train_margin(d)
        action = sample(margin, gen)
        reward = (action == best_action(x)).float()
        rewards.append(reward.mean().item())
        old, _ = dp.log_prob(margin, action)
        ref, _ = dp.log_prob(start, action)
        for _ in range(3):  # rounds on one set of samples, as far as the clip lets them go
            r = dp.policy_loss(model.train_margin(d), action, old, reward - reward.mean(), ref_log_prob=ref, kl=0.01,
                               hess=True)
            model.boost(d, step, r.grad, r.hess)
            step += 1
    return rewards[0], rewards[-1]


def main(argv=None) -> dict:
    p = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    p.add_argument("--rows", type=int, default=20000)
    p.add_argument("--rounds", type=int, default=30)
    a = p.parse_args(argv)
    out = {}
    for name, run, what in (("rank", rank, f"loss (from ln 2 = {math.log(2):.4f})"),
                            ("episodes", episodes, "probability of the paying action"),
                            ("policy", policy, "mean reward of sampled actions")):
        out[name] = run(a.rows, a.rounds)
        print(f"{name:9s} {what}: {out[name][0]:.4f} -> {out[name][1]:.4f}")
    return out


if __name__ == "__main__":
    main()
