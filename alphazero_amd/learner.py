"""The SGD step of the reference (training/nn_trainer.py:49-94) on batches that already live on the GPU
(SURVEY.md 8f-3).  Stock PyTorch: loss = -(pi * log_softmax(p)).sum(1).mean() + mse(v.squeeze(), z.squeeze())."""
from __future__ import annotations

import torch


def calculate_loss(model: torch.nn.Module, states, target_policies, target_values):
    pred_policies, pred_values = model(states)
    log_policies = torch.log_softmax(pred_policies, dim=1)
    policy_loss = -torch.sum(target_policies * log_policies, dim=1).mean()
    value_loss = torch.nn.functional.mse_loss(pred_values.squeeze(), target_values.squeeze())
    return policy_loss + value_loss, policy_loss.detach(), value_loss.detach()


def train_step(model: torch.nn.Module, optim: torch.optim.Optimizer, pool, batch_size: int = 64):
    """one Trainer.train(): zero_grad, loss on pool.sample(batch_size), backward, step"""
    batch = pool.sample(batch_size, timeout=1.0)
    if batch is None:
        raise ValueError("the experience pool holds no data")
    dev = next(model.parameters()).device
    states, pis, zs = (t.to(dev) for t in batch)
    model.train()
    optim.zero_grad()
    loss, pl, vl = calculate_loss(model, states, pis, zs)
    loss.backward()
    optim.step()
    model.eval()
    return float(loss.detach()), float(pl), float(vl)


class Muon(torch.optim.Optimizer):
    """Momentum whose update is orthogonalised (ops.orthogonalize) for every parameter of two or more dimensions, taken as the matrix
    (shape[0], rest); parameters of one dimension (biases, norms) take AdamW steps.  The reference trains with Adam
    (training/nn_trainer.py:36-94).  Parameters live on the GPU; all matrices of a type go through one call per step.

        buf <- lerp(buf, g, 1 - momentum);  u = lerp(g, buf, momentum) (nesterov) or buf
        p <- (1 - lr weight_decay) p - lr sqrt(max(1, rows / cols)) orthogonalize(u)"""

    def __init__(self, params, lr: float = 0.02, momentum: float = 0.95, nesterov: bool = True, steps: int = 5, weight_decay: float = 0.0,
                 adam_lr: float = 1e-3, betas=(0.9, 0.999), adam_eps: float = 1e-8):
        if not (lr >= 0 and adam_lr >= 0 and weight_decay >= 0 and 0 <= momentum < 1 and 0 <= betas[0] < 1 and 0 <= betas[1] < 1):
            raise ValueError("Muon: lr, adam_lr and weight_decay >= 0; momentum and betas in [0, 1)")
        params = list(params)
        common = dict(weight_decay=weight_decay)
        groups = [dict(params=[p for p in params if p.dim() >= 2], kind="matrix", lr=lr, momentum=momentum, nesterov=nesterov, steps=steps, **common),
                  dict(params=[p for p in params if p.dim() < 2], kind="vector", lr=adam_lr, betas=tuple(betas), eps=adam_eps, **common)]
        super().__init__([g for g in groups if g["params"]], dict(lr=lr))

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            by_type: dict = {}
            for p in group["params"]:
                if p.grad is not None and p.numel():
                    by_type.setdefault((p.device, p.dtype), []).append(p)
            for ps in by_type.values():
                (self._matrices if group["kind"] == "matrix" else self._vectors)(group, ps)
        return loss

    def _matrices(self, group, ps) -> None:
        from .ops import orthogonalize

        grads = [p.grad for p in ps]
        for p in ps:
            if "momentum" not in self.state[p]:
                self.state[p]["momentum"] = torch.zeros_like(p)
        bufs = [self.state[p]["momentum"] for p in ps]
        m = group["momentum"]
        torch._foreach_lerp_(bufs, grads, 1 - m)
        us = torch._foreach_lerp(grads, bufs, m) if group["nesterov"] else bufs
        us = orthogonalize([u.reshape(u.shape[0], -1) for u in us], steps=group["steps"])
        if group["weight_decay"]:
            torch._foreach_mul_(ps, 1 - group["lr"] * group["weight_decay"])
        scale = [-group["lr"] * max(1.0, u.shape[0] / u.shape[1]) ** 0.5 for u in us]
        torch._foreach_mul_(us, scale)
        torch._foreach_add_(ps, [u.view(p.shape) for u, p in zip(us, ps)])

    def _vectors(self, group, ps) -> None:
        b1, b2 = group["betas"]
        for p in ps:
            st = self.state[p]
            if "step" not in st:
                st.update(step=0, exp_avg=torch.zeros_like(p), exp_avg_sq=torch.zeros_like(p))
            st["step"] += 1
        grads, avg, sq = [p.grad for p in ps], [self.state[p]["exp_avg"] for p in ps], [self.state[p]["exp_avg_sq"] for p in ps]
        torch._foreach_lerp_(avg, grads, 1 - b1)
        torch._foreach_mul_(sq, b2)
        torch._foreach_addcmul_(sq, grads, grads, 1 - b2)
        if group["weight_decay"]:
            torch._foreach_mul_(ps, 1 - group["lr"] * group["weight_decay"])
        den = torch._foreach_sqrt(sq)
        torch._foreach_div_(den, [(1 - b2 ** self.state[p]["step"]) ** 0.5 for p in ps])
        torch._foreach_add_(den, group["eps"])
        num = torch._foreach_div(avg, [1 - b1 ** self.state[p]["step"] for p in ps])
        torch._foreach_addcdiv_(ps, num, den, -group["lr"])


class DataParallelLearner:
    """``train_step`` on every rank's own batch with the gradients averaged across ranks (BASELINE
    config 5): one process per GPU, ``torch.distributed`` (backend "nccl" = RCCL over xGMI; "gloo" in the CPU tests).

    Gradients live in a few large flat buckets (parameters' ``.grad`` are views into them), filled in backward order;
    a bucket's all-reduce is launched asynchronously from the hook of its last gradient, so it runs under the rest of
    backward.  xGMI is point to point (7 links per GPU), a ring all-reduce is per-link bound, so buckets are sized in
    tens of MB (few, large collectives): the reference nets (< 1 MB of gradients) go out as ONE collective.
    The reference has no counterpart: its learner is one process (training/nn_trainer.py:36-94)."""

    def __init__(self, model: torch.nn.Module, optim: torch.optim.Optimizer, bucket_bytes: int = 32 << 20,
                 process_group=None, force_collectives: bool = False):
        """force_collectives: run the hook / all-reduce path even with one rank (a process group must be initialised):
        how a one-GPU box exercises the code every rank of an N-GPU job runs."""
        import torch.distributed as dist

        self.model, self.optim, self.group = model, optim, process_group
        self.world = dist.get_world_size(process_group) if dist.is_initialized() else 1
        self.collective = self.world > 1 or (force_collectives and dist.is_initialized())
        params = [p for p in model.parameters() if p.requires_grad]
        self.buckets: list[torch.Tensor] = []
        self._bucket_of: dict[int, int] = {}
        self._need: list[int] = []
        cur: list[torch.nn.Parameter] = []
        cur_n = 0

        def close():
            nonlocal cur, cur_n
            if not cur:
                return
            flat = torch.zeros(cur_n, dtype=cur[0].dtype, device=cur[0].device)
            off = 0
            for p in cur:
                p.grad = flat[off:off + p.numel()].view_as(p)
                self._bucket_of[id(p)] = len(self.buckets)
                off += p.numel()
            self.buckets.append(flat)
            self._need.append(len(cur))
            cur, cur_n = [], 0

        for p in reversed(params):  # backward produces gradients roughly in reverse registration order
            if cur and (cur_n * p.element_size() >= bucket_bytes or p.dtype != cur[0].dtype):
                close()
            cur.append(p)
            cur_n += p.numel()
        close()
        self._left = list(self._need)
        self._handles: list = []
        self._sent: list[bool] = [False] * len(self.buckets)
        self.collectives_issued = 0
        if self.collective:
            for p in params:
                p.register_post_accumulate_grad_hook(self._on_grad)

    def _send(self, b: int) -> None:
        import torch.distributed as dist

        self._sent[b] = True
        self.collectives_issued += 1
        self._handles.append(dist.all_reduce(self.buckets[b], op=dist.ReduceOp.SUM, group=self.group, async_op=True))

    def _on_grad(self, p: torch.nn.Parameter) -> None:
        b = self._bucket_of[id(p)]
        self._left[b] -= 1
        if self._left[b] == 0:
            self._send(b)

    def step(self, pool, batch_size: int = 64):
        """one data-parallel Trainer.train(): every rank samples its own batch_size rows from its own pool"""
        batch = pool.sample(batch_size, timeout=1.0)
        if batch is None:
            raise ValueError("the experience pool holds no data")
        dev = next(self.model.parameters()).device
        states, pis, zs = (t.to(dev) for t in batch)
        self.model.train()
        for flat in self.buckets:  # zero_grad that keeps the views
            flat.zero_()
        self._left = list(self._need)
        self._handles = []
        self._sent = [False] * len(self.buckets)
        loss, pl, vl = calculate_loss(self.model, states, pis, zs)
        loss.backward()
        if self.collective:
            # A bucket whose hooks did not all fire (a parameter that took no part in this step's graph: its gradient
            # stays zero) is reduced here, in bucket order, so that every rank issues every bucket exactly once per
            # step.  (As with any data-parallel scheme the SET of unused parameters must be the same on every rank.)
            for b in range(len(self.buckets)):
                if not self._sent[b]:
                    self._send(b)
            for h in self._handles:
                h.wait()
            if self.world > 1:
                for flat in self.buckets:
                    flat.div_(self.world)
        self.optim.step()
        self.model.eval()
        return float(loss.detach()), float(pl), float(vl)
