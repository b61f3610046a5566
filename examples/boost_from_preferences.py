"""Boosting from preferences and rewards.

A context x has K actions.  People have compared pairs of actions; a logging
policy has chosen actions.  Two boosted models come out of that:

1. a reward model: one score for each (context, action) row, boosted on the
   gradient of ``preference_loss`` over the compared rows;
2. a policy: K scores a context, boosted on the gradient of
   ``policy_loss_logits`` at the logged actions, with the reward model's scores
   as rewards and a KL term that keeps it near the logging policy.

Each round fits one tree (one a class for the policy) to the negative gradient
with ``WarpGBM``'s regression, as a boosted fit does with its residuals.

    python examples/boost_from_preferences.py
"""
import contextlib
import io
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from warpgbm_b200 import WarpGBM, objectives  # noqa: E402


def fit_tree(bins, residual, depth=4, num_bins=32):
    """One tree on the residual of every row; its prediction for the same rows."""
    model = WarpGBM(objective="regression", num_bins=num_bins, max_depth=depth, n_estimators=1, learning_rate=1.0,
                    min_child_weight=5)
    with contextlib.redirect_stdout(io.StringIO()):
        model.fit(bins, residual)
        return torch.from_numpy(model.predict(bins)).to(bins.device)


def make_task(contexts, features, actions, pairs, seed, num_bins=32):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(contexts, features, device="cuda", generator=gen)
    # the value of an action: smooth in the context, different for each action
    direction = torch.randn(actions, features, device="cuda", generator=gen) / features ** 0.5
    value = 2.0 * torch.tanh(x @ direction.t())
    bins = (torch.sigmoid(x * 1.6) * num_bins).clamp(0, num_bins - 1).to(torch.int8)
    # compared pairs of actions of one context, and which one people preferred
    where = torch.randint(0, contexts, (pairs,), device="cuda", generator=gen)
    first = torch.randint(0, actions, (pairs,), device="cuda", generator=gen)
    second = (first + 1 + torch.randint(0, actions - 1, (pairs,), device="cuda", generator=gen)) % actions
    p = torch.sigmoid(value[where, first] - value[where, second])
    swap = torch.rand(pairs, device="cuda", generator=gen) > p
    chosen = where * actions + torch.where(swap, second, first)
    rejected = where * actions + torch.where(swap, first, second)
    # rows (context, action): the context's bins and the action as one more feature each
    onehot = torch.eye(actions, device="cuda", dtype=torch.int8).repeat(contexts, 1)
    rows = torch.cat([bins.repeat_interleave(actions, 0), onehot], 1).contiguous()
    # a logging policy that hardly knows the values
    logged_scores = 0.3 * value + torch.randn(contexts, actions, device="cuda", generator=gen)
    taken = torch.multinomial(logged_scores.softmax(1), 1, generator=gen)[:, 0]
    return dict(bins=bins.contiguous(), rows=rows, value=value, chosen=chosen, rejected=rejected,
                logged_scores=logged_scores, taken=taken)


def boost_reward(task, rounds, rate=0.5):
    score = torch.zeros(task["rows"].shape[0], device="cuda")
    losses = []
    for _ in range(rounds):
        r = objectives.preference_loss(score, task["chosen"], task["rejected"], beta=1.0)
        losses.append(r.loss)
        score += rate * fit_tree(task["rows"], -r.grad_logp * task["chosen"].numel(), depth=6)
    return score, torch.stack(losses)


def boost_policy(task, score, rounds, rate=0.3):
    contexts, actions = task["value"].shape
    logged = objectives.label_logprobs(task["logged_scores"], task["taken"])
    reward = score.view(contexts, actions).gather(1, task["taken"][:, None])[:, 0]
    advantage = (reward - reward.mean()) / reward.std()
    logits = torch.zeros(contexts, actions, device="cuda")
    losses = []
    for _ in range(rounds):
        r = objectives.policy_loss_logits(logits, task["taken"], logged.logp, advantage, ref_logp=logged.logp,
                                          kl_coef=0.02, entropy_coef=0.01, clip_low=0.8, clip_high=4.0,
                                          grad_scale=float(contexts))
        losses.append(r.loss)
        for k in range(actions):
            logits[:, k] += rate * fit_tree(task["bins"], -r.grad_logits[:, k].contiguous())
    return logits, torch.stack(losses)


def main(contexts=4000, features=8, actions=4, pairs=40000, rounds=30, seed=0):
    task = make_task(contexts, features, actions, pairs, seed)
    score, reward_losses = boost_reward(task, rounds)
    agree = (score[task["chosen"]] > score[task["rejected"]]).float().mean()
    logits, policy_losses = boost_policy(task, score, rounds)
    mean = lambda scores: (scores.softmax(1) * task["value"]).sum(1).mean()  # noqa: E731
    out = dict(reward_loss_first=float(reward_losses[0]), reward_loss_last=float(reward_losses[-1]),
               pair_agreement=float(agree), policy_loss_first=float(policy_losses[0]),
               policy_loss_last=float(policy_losses[-1]), value_uniform=float(task["value"].mean()),
               value_logged=float(mean(task["logged_scores"])), value_boosted=float(mean(logits)))
    for k, v in out.items():
        print(f"{k:20s} {v:.4f}")
    return out


if __name__ == "__main__":
    main()
