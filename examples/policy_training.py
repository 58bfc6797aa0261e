"""Train a logic network as a policy: real-valued observations in, one of ``k`` actions out, a clipped policy loss with a KL
term to the initial policy.

    observation -> LogicLayerNorm -> sigmoid (soft bits) -> LogicLayer -> LogicDropout -> LogicLayer -> GroupSum -> logits

The task is a contextual bandit: the rewarded action is the one whose hidden direction the observation points along most.
Run ``python examples/policy_training.py [--steps N]`` on a machine with a B200.
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import compactlogic_b200 as cl  # noqa: E402


def build(features: int, width: int, actions: int, seed: int = 0) -> torch.nn.Sequential:
    torch.manual_seed(seed)
    model = torch.nn.Sequential(
        cl.LogicLayerNorm(features), torch.nn.Sigmoid(),
        cl.LogicLayer(features, width), cl.LogicDropout(0.05, rescale=False, seed=seed),
        cl.LogicLayer(width, width), cl.GroupSum(actions, tau=width / actions / 12.0)).cuda()
    return cl.fuse_groupsum(model)


def rollout(model, directions, n, generator):
    """Observations, the actions that the policy draws for them, their log-probabilities and rewards."""
    obs = torch.randn(n, directions.shape[1], device="cuda", generator=generator) * 2.0 + 0.5
    with torch.no_grad():
        logits = model(obs)  # in training mode: the soft network is the policy that learns
        actions = torch.multinomial(torch.softmax(logits.float(), 1), 1, generator=generator)[:, 0]
        old = cl.action_log_probs(logits, actions)
        best = ((obs - 0.5) @ directions.t()).argmax(1)
    return obs, actions, old, (actions == best).float()


def train(steps: int = 60, epochs: int = 3, n: int = 2048, features: int = 32, width: int = 2000, actions: int = 5,
          seed: int = 0, verbose: bool = True):
    """The mean reward of the first and of the last rollouts."""
    model, reference = build(features, width, actions, seed), build(features, width, actions, seed)
    for m in reference.modules():  # the same policy at the start, without the mask
        if isinstance(m, cl.LogicDropout):
            m.p = 0.0
    generator = torch.Generator(device="cuda").manual_seed(seed)
    directions = torch.randn(actions, features, device="cuda", generator=generator)
    opt = torch.optim.Adam(model.parameters(), lr=0.05)
    rewards = []
    for step in range(steps):
        obs, act, old, reward = rollout(model, directions, n, generator)
        with torch.no_grad():
            ref = cl.action_log_probs(reference(obs), act)
        advantage = (reward - reward.mean()) / (reward.std() + 1e-6)
        for _ in range(epochs):
            opt.zero_grad(set_to_none=True)
            out = cl.policy_loss(model(obs), act, advantage, old, ref_log_probs=ref, clip=0.2, kl_coef=0.002)
            out.loss.backward()
            opt.step()
        rewards.append(reward.mean())
        if verbose and step % 10 == 0:
            print(f"step {step:3d}  reward {reward.mean().item():.3f}  loss {out.loss.item():+.4f}  kl {out.kl.mean().item():.4f}")
    rewards = torch.stack(rewards).tolist()
    return sum(rewards[:3]) / 3, sum(rewards[-3:]) / 3


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--steps", type=int, default=60)
    first, last = train(ap.parse_args().steps)
    print(f"mean reward {first:.3f} -> {last:.3f}")
