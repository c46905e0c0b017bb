"""ActorCriticNet (/root/reference/go_ai/models/ac_net.py:8-64) on the HIP forward."""
import numpy as np
import torch

from . import AdamW, RLNet


def _legal_moves(states):
    """uint8 [n, A]: 1 where a move is allowed (plane 3 holds the invalid ones; the pass always is), as data.batch_valid_moves."""
    n = states.shape[0]
    board = (states[:, 3] == 0).view(n, -1)
    return torch.cat([board, board.new_ones((n, 1))], dim=1).view(torch.uint8)


class ActorCriticNet(RLNet):
    kind = "ac"

    def __init__(self, size, **kw):
        super().__init__(size, **kw)
        self.action_size = size * size + 1

    def move_logprobs(self, states, actions=None, top=0, temperature=1.0):
        """What the actor thinks of positions [n, 6, s, s] and of the moves that were played there (actions [n], -1: none): an
        engine.ActionLogprobs of GPU tensors over the legal moves -- log probabilities, entropy, lse, and the `top` moves it
        would rather play with theirs."""
        from ..engine import _dev_u8_states
        self._pull_trained()
        st = _dev_u8_states(states, self.ctx.device)
        logits = self.ctx.nn_forward(st)[0]
        return self.ctx.action_logprobs(logits, actions, valid=_legal_moves(st), temperature=temperature, top=top)

    def _policy_batch(self, states, actions, advantages, entropy_weight, temperature):
        """policy_step's arguments on the GPU: states, legal moves, actions, advantages."""
        from ..engine import _dev_u8_states
        dev = self.ctx.device
        shape = tuple(states.shape) if torch.is_tensor(states) else np.shape(states)
        if len(shape) != 4 or shape[1:] != (6, self.size, self.size):
            raise ValueError(f"policy_step: states of shape {shape}, expected (n, 6, {self.size}, {self.size})")
        st = _dev_u8_states(states if torch.is_tensor(states) else np.asarray(states), dev)
        n = st.shape[0]
        if n < 2:
            raise ValueError(f"policy_step: {n} position(s); BatchNorm needs at least 2")
        if not (1e-4 <= temperature <= 1e4 and np.isfinite(entropy_weight)):
            raise ValueError(f"policy_step: temperature {temperature} (1e-4 .. 1e4), entropy_weight {entropy_weight} (finite)")
        actions = torch.as_tensor(np.asarray(actions) if not torch.is_tensor(actions) else actions)
        adv = torch.as_tensor(np.asarray(advantages, dtype=np.float32) if not torch.is_tensor(advantages) else advantages.detach())
        adv = adv.to(dev, dtype=torch.float32)
        if actions.shape != (n,) or adv.shape != (n,):
            raise ValueError(f"policy_step: {n} positions, actions of shape {tuple(actions.shape)}, advantages of shape {tuple(adv.shape)}")
        actions = self.ctx._per_row(actions, n, torch.int32, "policy_step: actions")
        valid = _legal_moves(st)
        at = actions.clamp(0, self.action_size - 1).long()[:, None]
        illegal = (actions >= 0) & (valid.gather(1, at)[:, 0] == 0)
        wrong = torch.stack([(actions >= self.action_size).any(), illegal.any(), ~torch.isfinite(adv).all()]).tolist()
        if wrong[0]:
            raise ValueError(f"policy_step: actions beyond the board's {self.action_size}")
        if wrong[1]:
            raise ValueError("policy_step: actions that are not legal in their position")
        if wrong[2]:
            raise ValueError("policy_step: advantages that are not finite")
        return st, valid, actions, adv

    def policy_step(self, optimizer, states, actions, advantages, entropy_weight=0.01, temperature=1.0):
        """One policy-gradient step of the actor and the trunk on n >= 2 positions: the loss is
            -mean(advantages * log p[actions]) - entropy_weight * mean(entropy)
        over the legal moves; actions [n]: legal ones, -1: none (the position counts in the entropy alone); optimizer: an AdamW (the
        critic's head has no gradient and stays as it is).  Returns (loss, mean log probability of the actions, mean entropy)
        from before the step."""
        if not isinstance(optimizer, AdamW):
            raise ValueError("policy_step: the optimizer must be a go_ai.models.AdamW")
        # all checks come before anything moves: parameters, moments, BatchNorm statistics, the training buffers
        entropy_weight, temperature = float(entropy_weight), float(temperature)
        st, valid, actions, adv = self._policy_batch(states, actions, advantages, entropy_weight, temperature)
        self._check_optimizer(optimizer)
        n = st.shape[0]
        if n > self.train_batch:
            self._grow_train_batch(n)
        self.train()
        dev = self._train.device
        self._bind_optimizer(optimizer)
        self._train_dirty = True
        logits = self._train.train_actor_forward(st)
        lp = self._train.action_logprobs(logits, actions, valid=valid, temperature=temperature)
        d_entropy = torch.full((n,), -entropy_weight / n, dtype=torch.float32, device=dev)
        d_logits = self._train.action_logprobs_grad(logits, actions, lp.lse, lp.entropy, adv * (-1.0 / n), d_entropy, valid=valid,
                                                    temperature=temperature, out=logits)
        self._train.train_actor_backward(d_logits)
        optimizer.step([None if k.startswith("crit_head.") else g for k, g in zip(optimizer._net_names, optimizer._net_grads)])
        stats = torch.stack([-(adv * lp.logp).mean() - entropy_weight * lp.entropy.mean(), lp.logp.mean(), lp.entropy.mean()])
        return tuple(stats.tolist())
