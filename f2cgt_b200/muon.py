"""Muon for the weight matrices of a network: momentum, and updates whose singular values are all about one.

The step itself is ``ops.muon_step``: one launch for all matrices up to 128 x 256 (or transposed), 17 launches for those of each larger
shape.  A GraphSAGE network of 128 columns takes 53 us, one of 256 columns 185.  What is no matrix (biases) is updated by Adam, in the
fused kernel ``train_graphsage.DirectFusedAdam`` calls.  Like that class it is a plain object: ``step()``, ``zero_grad()``, ``lr``.
"""
import torch

from . import ops


def _adam_step(adam):
    """``DirectFusedAdam.step`` for a torch that does not expose the fused kernel."""
    (beta1, beta2), count = adam.betas, adam.steps[0].add_(1)
    for p, m, v in zip(adam.params, adam.exp_avg, adam.exp_avg_sq):
        m.lerp_(p.grad, 1 - beta1)
        v.mul_(beta2).addcmul_(p.grad, p.grad, value=1 - beta2)
        p.sub_(m / (1 - beta1 ** count) * adam.lr / ((v / (1 - beta2 ** count)).sqrt() + adam.eps))


class Muon:
    """``params``: parameters on one device; matrices (float32, float16 or bfloat16) are orthogonalised, the others (float32) go to Adam with
    ``adam_lr``, which moves with ``lr`` (a schedule sets ``lr`` alone; of ``lr=0`` there is no ratio to keep, and Adam's rate stays ``adam_lr``).
    ``lr`` times ``sqrt(max(1, rows / cols))`` is the size of an update's singular values.  Momenta are float32.
    Matrices without a gradient are left alone."""

    def __init__(self, params, lr=0.02, momentum=0.95, nesterov=True, weight_decay=0.0, steps=5, coefficients=ops.NEWTON_SCHULZ, eps=1e-7,
                 adam_lr=0.003):
        from .train_graphsage import DirectFusedAdam
        params = [p for p in params if p.requires_grad]
        self.matrices = [p for p in params if p.dim() == 2]
        for p in self.matrices:
            if not p.is_cuda or not p.is_contiguous() or p.dtype not in (torch.float32, torch.float16, torch.bfloat16):
                raise RuntimeError("Muon: matrices must be contiguous CUDA tensors of float32, float16 or bfloat16")
        self.momenta = [torch.zeros_like(p, dtype=torch.float32) for p in self.matrices]
        self.momentum, self.nesterov, self.weight_decay = float(momentum), bool(nesterov), float(weight_decay)
        self.steps, self.coefficients, self.eps = int(steps), coefficients, float(eps)
        others = [p for p in params if p.dim() != 2]
        self.adam = DirectFusedAdam(others, lr=adam_lr) if others else None
        self._lr, self._adam_ratio = float(lr), float(adam_lr) / float(lr) if lr else None

    @property
    def lr(self):
        return self._lr

    @lr.setter
    def lr(self, value):  # a schedule moves both learning rates
        self._lr = float(value)
        if self.adam is not None and self._adam_ratio is not None:
            self.adam.lr = self._lr * self._adam_ratio

    def zero_grad(self, set_to_none=True):
        for p in self.matrices:
            if set_to_none:
                p.grad = None
            elif p.grad is not None:
                p.grad.zero_()
        if self.adam is not None:
            self.adam.zero_grad(set_to_none)

    @torch.no_grad()
    def step(self):
        by_type = {}
        for p, m in zip(self.matrices, self.momenta):
            if p.grad is not None:
                by_type.setdefault(p.dtype, []).append((p, p.grad if p.grad.is_contiguous() else p.grad.contiguous(), m))
        for group in by_type.values():
            weights, grads, momenta = zip(*group)
            ops.muon_step(weights, grads, momenta, self._lr, self.momentum, self.nesterov, self.weight_decay, self.steps, self.coefficients, self.eps)
        if self.adam is not None and any(p.grad is not None for p in self.adam.params):
            if any(p.grad is None for p in self.adam.params):
                raise RuntimeError("Muon: the parameters that are no matrices are updated together: one of them has no gradient")
            if self.adam.available():
                self.adam.step()
            else:
                _adam_step(self.adam)

    def state_dict(self):
        state = dict(lr=self._lr, momenta=self.momenta)
        if self.adam is not None:
            state.update(adam_lr=self.adam.lr, adam_ratio=self._adam_ratio, exp_avg=self.adam.exp_avg, exp_avg_sq=self.adam.exp_avg_sq, adam_steps=self.adam.steps[0])
        return state

    def load_state_dict(self, state):
        pairs = list(zip(self.momenta, state["momenta"]))
        if len(state["momenta"]) != len(self.momenta):
            raise RuntimeError("Muon: the state is of another network")
        if self.adam is not None:
            pairs += list(zip(self.adam.exp_avg, state["exp_avg"])) + list(zip(self.adam.exp_avg_sq, state["exp_avg_sq"]))
            pairs.append((self.adam.steps[0], state["adam_steps"]))
        for mine, given in pairs:
            if mine.shape != given.shape:
                raise RuntimeError("Muon: the state is of another network")
        for mine, given in pairs:
            mine.copy_(given)
        self.lr = state["lr"]
        if self.adam is not None and "adam_lr" in state:  # (states of before have no rate of Adam's)
            self.adam.lr, self._adam_ratio = float(state["adam_lr"]), state["adam_ratio"]
