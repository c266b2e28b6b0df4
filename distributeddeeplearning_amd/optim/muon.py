"""Muon over the flat arenas (kernels K22 / K23): momentum whose direction is orthogonalised per weight matrix.

Every parameter of two or more dimensions is a matrix ``[out, rest]`` (a convolution filter: ``[Cout, Cin * R * S]``; the
order of its columns, KRSC in memory, does not change the result).  Vectors - BatchNorm, biases - take plain momentum SGD.

Update rule for matrices: ``v = mu*v + g``; ``u = g + mu*v`` (nesterov) or ``v``; ``O = orthogonalize(u)``
(:func:`distributeddeeplearning_amd.ops.functional.orthogonalize`); ``w = w*(1 - lr*wd) - lr*sqrt(max(1, out/rest))*O``.
For vectors: the rule of ``FusedSGD`` with ``vector_lr_scale*lr``.

The reference has plain momentum SGD only (``imagenet_pytorch_horovod.py:333``); a third optimizer next to ``FusedSGD`` and
``FusedLARS``, with the same arenas, checkpoints, launch tape and learning-rate handling.  All matrices of a step share the
launches of their form (up to 64 matrices a call).  Their products are those of ``orthogonalize``: 16-bit operands above 32 rows,
for fp32 parameters too.  Like ``FusedLARS`` it updates after the last gradient bucket: a bucket at a time would
leave the products of a few matrices alone on the chip.  Every rank orthogonalises every matrix, in a fixed order: replicas
stay equal bit for bit.
"""
from __future__ import annotations

import math

import torch

from ..ops import functional as ops
from .fused import _ArenaOptimizer

__all__ = ["FusedMuon"]


class FusedMuon(_ArenaOptimizer):
    def __init__(self, named_parameters, lr=0.02, momentum=0.95, weight_decay=0.0, nesterov=True, steps=5,
                 coefficients=ops.ORTHO_COEFFICIENTS, eps=1e-7, vector_lr_scale=1.0, weight_decay_filter=None,
                 engine_config=None):
        if lr < 0 or momentum < 0 or weight_decay < 0 or vector_lr_scale < 0:
            raise ValueError("negative hyper-parameter")
        ops._check_steps(steps, coefficients, eps)
        named = list(named_parameters)
        self._refuse_sizes(named)
        a, b, c = (float(v) for v in coefficients)
        defaults = dict(lr=lr, momentum=momentum, weight_decay=weight_decay, nesterov=nesterov, steps=steps,
                        ortho_a=a, ortho_b=b, ortho_c=c, eps=eps, vector_lr_scale=vector_lr_scale)
        super().__init__(named, defaults, weight_decay_filter, engine_config)
        self._vector_lr = None            # (frozen learning rate: the vectors')
        # matrices of one arena and one decay flag, in calls of at most ortho_max_groups
        self._matrices = []
        for dt in self.arena.plans:
            for decay in (False, True):
                segs = [s for r in self.runs if r["adapt"] and r["dtype"] == dt and r["decay"] == decay
                        for s in r["segments"] if s.numel > 0]
                if segs:
                    self._matrices.append({"dtype": dt, "decay": decay, "segments": segs, "calls": None})

    @staticmethod
    def _refuse_sizes(named):
        """Refuses a matrix that the kernels do not take, before the parameters are moved into the arenas."""
        from ..ops import kernels

        for entry in named:
            p = entry[1] if isinstance(entry, tuple) else entry
            if p.is_cuda and p.requires_grad and p.dim() > 1 and p.numel() > 0 and kernels.enabled():
                kernels.ortho_workspace_of(((p.shape[0], p.numel() // p.shape[0], 1),))

    def _hip(self):
        from ..ops import kernels

        return self.arena.device.type == "cuda" and kernels.enabled()

    def _tables(self, entry):
        if entry["calls"] is None:
            from ..ops import kernels

            rows = [(0, s.offset, 0, 0, 0, 0, 0, 0, s.shape[0], s.numel // s.shape[0], 1) for s in entry["segments"]]
            per = kernels.ortho_max_groups()
            tables = [kernels.ortho_table(rows[k:k + per]) for k in range(0, len(rows), per)]
            entry["calls"] = [(t, n, {}) for t, n in tables]
        return entry["calls"]

    @staticmethod
    def _workspace(table, count, known, coefficients, steps):
        """Bytes of a call's workspace (``known``: what earlier steps found)."""
        from ..ops import kernels

        key = (coefficients, steps)
        if key not in known:
            known[key] = kernels.ortho_workspace(table, count, coefficients, steps)
        return known[key]

    # the vectors' rate is a device scalar of its own: lr * vector_lr_scale is rounded to fp32 once, as where it is passed by value
    def freeze_lr(self):
        out = super().freeze_lr()
        if self._vector_lr is None:
            self._vector_written = self._vector_rate()
            self._vector_lr = torch.full((1,), self._vector_written, dtype=torch.float32, device=self.arena.device)
        return out

    def sync_lr(self):
        super().sync_lr()
        if self._vector_lr is not None and self._vector_rate() != self._vector_written:
            self._vector_written = self._vector_rate()
            self._vector_lr.fill_(self._vector_written)

    def _vector_rate(self):
        return float(self.param_groups[0]["lr"]) * self.param_groups[0]["vector_lr_scale"]

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        hip = self._hip()
        if hip:
            from ..ops import hip_ops

            with hip_ops._on(self.arena.device):
                self._update(hip)
        else:
            self._update(hip)
        self._step += 1
        self._notify_weights_changed(hip)
        return loss

    def _update(self, hip):
        from ..ops import kernels

        g0 = self.param_groups[0]
        lr, mu, wd, nesterov = g0["lr"], g0["momentum"], g0["weight_decay"], g0["nesterov"]
        steps, coefficients, eps = g0["steps"], (g0["ortho_a"], g0["ortho_b"], g0["ortho_c"]), g0["eps"]
        ops._check_steps(steps, coefficients, eps)        # (the group's values may have been changed)
        klr, kscale = self._kernel_lr(lr)
        for entry in self._matrices:
            dt, run_wd = entry["dtype"], wd if entry["decay"] else 0.0
            w, g, v = self._weights(dt), self.arena.grads[dt], self.momentum_buf[dt]
            if hip:
                lowp = self.arena.params[dt] if dt in self.master else None
                for table, count, known in self._tables(entry):
                    nbytes = self._workspace(table, count, known, coefficients, steps)
                    work = torch.empty(nbytes, dtype=torch.uint8, device=w.device) if nbytes else None
                    kernels.muon_step_(table, count, w, g, v, lowp, klr, mu, run_wd, nesterov, kscale, coefficients,
                                       steps, eps, work)
                continue
            for s in entry["segments"]:
                sl = slice(s.offset, s.offset + s.numel)
                grad = g[sl].to(torch.float32)
                v[sl].mul_(mu).add_(grad)
                u = grad.add(v[sl], alpha=mu) if nesterov else v[sl]
                rows = s.shape[0]
                o = ops.orthogonalize_plain(u.view(rows, -1), steps, coefficients, eps)
                scale = math.sqrt(max(1.0, rows / (s.numel // rows)))
                w[sl].mul_(1.0 - lr * run_wd).sub_(o.reshape(-1), alpha=lr * scale)
                self._publish(dt, s.offset, s.offset + s.numel)
        for run in self.runs:
            if run["adapt"]:
                continue
            dt, a, b = run["dtype"], run["start"], run["end"]
            run_wd = wd if run["decay"] else 0.0
            w, g, v = self._weights(dt)[a:b], self.arena.grads[dt][a:b], self.momentum_buf[dt][a:b]
            if hip:
                lowp = self.arena.params[dt][a:b] if dt in self.master else None
                rate = self._vector_rate() if kscale is None else self._frozen_lr
                kernels.fused_sgd_(w, g, v, lowp, rate, mu, run_wd, nesterov, None if kscale is None else self._vector_lr)
                continue
            grad = g.to(torch.float32)
            if run_wd:
                grad = grad.add(w, alpha=run_wd)
            v.mul_(mu).add_(grad)
            w.add_(grad.add(v, alpha=mu) if nesterov else v, alpha=-self._vector_rate())
            self._publish(dt, a, b)
