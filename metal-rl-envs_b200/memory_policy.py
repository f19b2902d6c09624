"""A policy with memory, trained by gradient on the batched environments: CartPole with its velocities
hidden, which no memoryless policy solves (one frame does not say which way the pole falls).

The policy's layers are this package's operators: a linear attention over the episode so far
(linear_attention: `step` when acting, `attend` over the collected trajectory), a gated feed-forward block
(gated_ffn.apply) and plain matrix products between them; adamw.step trains it. One update steps N
environments T times (cartpole_metal.step), keeping each environment's attention state from update to
update, then runs the same T x N tokens through the trajectory form and takes one actor-critic step
(Williams 1992's REINFORCE with a learned baseline). The environments' `dones` cut the memory at episode ends.

    python memory_policy.py --envs 1024 --steps 64 --updates 150

The reference trains memoryless MLPs (es.py) and has no counterpart of this module.
"""

import argparse
from dataclasses import dataclass

import torch

import adamw
import cartpole_metal
import gated_ffn
import linear_attention
import rlenv_lib as _rl

OBSERVED = (0, 2)  # cart position and pole angle; the velocities stay hidden


@dataclass
class Config:
    envs: int = 1024
    steps: int = 64          # environment steps an update
    updates: int = 150
    heads: int = 4
    width: int = 16          # of a head
    hidden: int = 128        # of the gated block
    lr: float = 3e-3
    discount: float = 0.98
    entropy: float = 0.01
    max_norm: float = 1.0    # of the gradient
    state_bits: int = 32     # of the optimizer's moments
    seed: int = 0


class MemoryPolicy:
    """tokens (..., features) -> action logits and value. Parameters are float32 leaves in `parameters`."""

    def __init__(self, cfg, features=len(OBSERVED) + 1, actions=2):
        self.cfg = cfg
        dev, model = _rl.device(), cfg.heads * cfg.width
        g = torch.Generator(device=dev).manual_seed(cfg.seed)

        def leaf(rows, cols, gain=1.0):
            w = torch.randn((rows, cols), generator=g, device=dev) * gain * rows ** -0.5
            return w.requires_grad_()

        self.embed = leaf(features, model)
        self.qkv = leaf(model, 3 * model)
        self.mix = leaf(model, model)
        self.gate, self.up, self.down = leaf(model, cfg.hidden), leaf(model, cfg.hidden), leaf(cfg.hidden, model)
        self.head = leaf(model, actions + 1, 0.1)
        self.parameters = [self.embed, self.qkv, self.mix, self.gate, self.up, self.down, self.head]
        # memories of about 2, 4, 8, .. steps
        self.decay = 1.0 - 0.5 ** (1.0 + torch.arange(cfg.heads, device=dev, dtype=torch.float32))

    def fresh_state(self, n):
        c = self.cfg
        return torch.zeros((n, c.heads, c.width, c.width), device=self.decay.device)

    def _split(self, x):
        """q, k, v (..., H, D) as views of one product."""
        qkv = (_normal(x) @ self.qkv).unflatten(-1, (3, self.cfg.heads, self.cfg.width))
        return qkv.unbind(-3)

    def _rest(self, x, out):
        x = x + out.flatten(-2) @ self.mix
        x = x + gated_ffn.apply(_normal(x), self.gate, self.up, "silu") @ self.down
        y = _normal(x) @ self.head
        return y[..., :-1], y[..., -1]

    @torch.no_grad()
    def act(self, tokens, state, resets):
        """One token for every environment, tokens (N, features); state (N, H, D, D) is updated in place."""
        x = tokens @ self.embed
        return self._rest(x, linear_attention.step(*self._split(x), self.decay, state, resets))

    def trajectory(self, tokens, state, resets):
        """Logits (T, N, actions) and values (T, N) of T tokens, differentiable in the parameters."""
        x = tokens @ self.embed
        out, _ = linear_attention.attend(*self._split(x), self.decay, state, resets)
        return self._rest(x, out)


def _normal(x):
    """Root-mean-square normalisation."""
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6)


def observe(state):
    """(N, features) tokens of CartPole states (4, N): what is observed, scaled to order one, and a one."""
    seen = state[list(OBSERVED)] * torch.tensor([[1.0], [10.0]], device=state.device)
    return torch.cat([seen, torch.ones_like(seen[:1])]).t()


@dataclass
class Rollout:
    tokens: torch.Tensor   # (T, N, features)
    actions: torch.Tensor  # (T, N)
    rewards: torch.Tensor  # (T, N)
    dones: torch.Tensor    # (T, N)
    resets: torch.Tensor   # (T, N): tokens that start an episode
    memory: torch.Tensor   # (N, H, D, D): the attention state before the first token
    logits: torch.Tensor   # (T, N, actions), as acted on


def collect(policy, env_state, memory, resets, steps, generator):
    """(Rollout, env_state, memory, resets) after `steps` steps of every environment."""
    start = memory.clone()
    tokens, actions, rewards, dones, first, logits = [], [], [], [], resets, []
    for _ in range(steps):
        x = observe(env_state)
        y, _ = policy.act(x, memory, resets)
        a = torch.multinomial(torch.softmax(y, -1), 1, generator=generator)[:, 0]
        env_state, reward, done = cartpole_metal.step(env_state, a)
        for kept, new in ((tokens, x), (actions, a), (rewards, reward), (dones, done), (logits, y)):
            kept.append(new)
        resets = done
    dones = torch.stack(dones)
    return Rollout(torch.stack(tokens), torch.stack(actions), torch.stack(rewards), dones,
                   linear_attention.episode_starts(dones, first), start, torch.stack(logits)), env_state, memory, resets


def returns_of(rewards, dones, values, discount):
    """Discounted returns (T, N), cut at episode ends, the last step's continued by its value."""
    out, ahead = torch.empty_like(rewards), values[-1]
    for t in range(rewards.shape[0] - 1, -1, -1):
        ahead = rewards[t] + discount * torch.where(dones[t], 0.0, ahead)
        out[t] = ahead
    return out


def update(policy, optimizer, rollout):
    """One actor-critic step on a rollout; returns the loss."""
    cfg = policy.cfg
    logits, values = policy.trajectory(rollout.tokens, rollout.memory, rollout.resets)
    returns = returns_of(rollout.rewards, rollout.dones, values.detach(), cfg.discount)
    gain = returns - values.detach()
    gain = (gain - gain.mean()) / (gain.std() + 1e-6)
    logp = torch.log_softmax(logits, -1)
    chosen = logp.gather(-1, rollout.actions[..., None].long())[..., 0]
    entropy = -(logp.exp() * logp).sum(-1).mean()
    loss = -(gain * chosen).mean() + 0.5 * torch.nn.functional.smooth_l1_loss(values, returns) - cfg.entropy * entropy
    grads = torch.autograd.grad(loss, policy.parameters)
    norm = torch.stack([g.square().sum() for g in grads]).sum().sqrt()
    with torch.no_grad():
        adamw.step(policy.parameters, list(grads), optimizer, lr=cfg.lr, weight_decay=0.0,
                   grad_scale=torch.clamp(cfg.max_norm / (norm + 1e-6), max=1.0))
    return loss.detach()


def train(cfg, log=lambda *_: None):
    """Trains a policy; returns (policy, mean episode length at each update). log(update, mean length, loss)
    is called after every update."""
    policy = MemoryPolicy(cfg)
    optimizer = adamw.init_state(policy.parameters, cfg.state_bits, seed=cfg.seed)
    dev = policy.decay.device
    generator = torch.Generator(device=dev).manual_seed(cfg.seed)
    cartpole_metal.reseed(cfg.seed)
    env_state, memory = cartpole_metal.reset(cfg.envs), policy.fresh_state(cfg.envs)
    resets = torch.ones(cfg.envs, dtype=torch.bool, device=dev)
    lengths = []
    for i in range(cfg.updates):
        rollout, env_state, memory, resets = collect(policy, env_state, memory, resets, cfg.steps, generator)
        loss = update(policy, optimizer, rollout)
        # steps an episode end, over the rollout
        lengths.append(rollout.dones.numel() / max(1.0, rollout.dones.sum().item()))
        log(i + 1, lengths[-1], loss.item())
    return policy, lengths


def main(argv=None):
    parser = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    for name, value in vars(Config()).items():
        parser.add_argument(f"--{name.replace('_', '-')}", type=type(value), default=value)
    cfg = Config(**vars(parser.parse_args(argv)))
    train(cfg, lambda i, length, loss: print(f"update {i:4d} | {length:8.1f} steps an episode end | loss {loss:8.4f}",
                                             flush=True))
    return 0


if __name__ == "__main__":
    main()
