"""Optimizers over the engine's flat buckets.

The reference's server-side SGD aggregation (PS path) and per-rank
``apply_gradients`` (Horovod path) collapse to: every rank applies the
identical update to the identical averaged gradients.

``FlatSGD`` walks the DataParallel engine's buckets and updates each flat
param/grad pair with ONE fused HIP kernel launch per bucket
(sgd_momentum_flat: wd + momentum + nesterov + lr in a single pass,
fp32 momentum for bf16 params).  Torch fallback keeps CPU tests running.
``FlatAdam`` is the BERT-path equivalent (fused adamw_flat kernel).
``FlatMuon`` orthogonalises the momentum of hidden matrices (all of a shape
in one batch of Newton-Schulz products) and runs AdamW on everything else.
"""

from __future__ import annotations

from typing import Dict, List, Optional, Tuple

import torch

from ..ops import functional as F_amd
from ..ops import native, native_available
from .ddp import DataParallel


class _FlatOptimBase:
    def __init__(self, engine: DataParallel):
        self.engine = engine
        self.buckets = engine.plan.buckets
        # one contiguous param mirror per bucket so the fused kernel walks
        # a single pointer; params are re-viewed into it (zero-copy update).
        self.flat_params: List[torch.Tensor] = []
        # fp32 master weights for reduced-precision params (bf16 training):
        # the fused kernels update the master and write the bf16 copy.
        self.masters: List[Optional[torch.Tensor]] = []
        for b in self.buckets:
            flat_p = torch.empty_like(b.flat)
            off = 0
            with torch.no_grad():
                for p in b.params:
                    flat_p[off:off + p.numel()].copy_(p.detach().reshape(-1))
                    # re-point the parameter at its slice of the flat buffer
                    p.data = flat_p[off:off + p.numel()].view_as(p)
                    off += p.numel()
            self.flat_params.append(flat_p)
            self.masters.append(flat_p.float()
                                if flat_p.dtype != torch.float32 else None)

    def zero_grad(self) -> None:
        self.engine.zero_grad()

    def refresh_masters(self) -> None:
        """Re-derive fp32 master weights from the (bf16) params.

        Needed after ``model.load_state_dict`` — loading copies into the
        flat param buffers, leaving masters captured at construction time
        stale.  Checkpoints that carry optimizer state overwrite these
        again in ``load_state_dict`` (SURVEY.md §6.4 resume contract).
        """
        for fp, master in zip(self.flat_params, self.masters):
            if master is not None:
                master.copy_(fp.float())

    def state_dict(self) -> dict:
        raise NotImplementedError

    def load_state_dict(self, sd: dict) -> None:
        raise NotImplementedError


class FlatSGD(_FlatOptimBase):
    def __init__(self, engine: DataParallel, lr: float = 0.1,
                 momentum: float = 0.9, weight_decay: float = 1e-4,
                 nesterov: bool = False):
        super().__init__(engine)
        self.lr, self.momentum = lr, momentum
        self.weight_decay, self.nesterov = weight_decay, nesterov
        self.momentum_bufs = [
            torch.zeros(fp.numel(), dtype=torch.float32, device=fp.device)
            for fp in self.flat_params]

    @torch.no_grad()
    def step(self) -> None:
        for fp, b, mbuf, master in zip(self.flat_params, self.buckets,
                                       self.momentum_bufs, self.masters):
            g = b.flat
            if fp.is_cuda and native_available():
                if master is not None:
                    native().sgd_momentum_flat_master(
                        fp, g, mbuf, master, self.lr, self.momentum,
                        self.weight_decay, self.nesterov)
                else:
                    native().sgd_momentum_flat(
                        fp, g, mbuf, self.lr, self.momentum,
                        self.weight_decay, self.nesterov)
                continue
            # torch fallback — numerically the reference update:
            # m = mu*m + (g + wd*p); p -= lr * (m or g+mu*m)
            pv = master if master is not None else fp
            g32 = g.float()
            if self.weight_decay:
                g32 = g32.add(pv.float(), alpha=self.weight_decay)
            mbuf.mul_(self.momentum).add_(g32)
            upd = g32.add(mbuf, alpha=self.momentum) if self.nesterov else mbuf
            if master is not None:
                master.sub_(self.lr * upd)
                fp.copy_(master.to(fp.dtype))
            else:
                fp.copy_((fp.float() - self.lr * upd).to(fp.dtype))

    def state_dict(self) -> dict:
        return {"momentum_bufs": self.momentum_bufs, "masters": self.masters,
                "lr": self.lr, "momentum": self.momentum,
                "weight_decay": self.weight_decay, "nesterov": self.nesterov}

    def load_state_dict(self, sd: dict) -> None:
        for dst, src in zip(self.momentum_bufs, sd["momentum_bufs"]):
            dst.copy_(src.to(dst.device))
        for dst, src in zip(self.masters, sd.get("masters", [])):
            if dst is not None and src is not None:
                dst.copy_(src.to(dst.device))
        self.lr = sd["lr"]
        self.momentum = sd["momentum"]
        self.weight_decay = sd["weight_decay"]
        self.nesterov = sd["nesterov"]


class _FlatAdamBase(_FlatOptimBase):
    """Counts steps on the parameters' device, so that a captured step that
    is replayed counts (and corrects its moments' bias) like an eager one."""

    def __init__(self, engine: DataParallel):
        super().__init__(engine)
        device = self.flat_params[0].device if self.flat_params else "cpu"
        self._steps = torch.zeros((), dtype=torch.int64, device=device)
        # 1 / (1 - beta ** t) of both betas
        self._inverse = torch.ones(2, dtype=torch.float32, device=device)

    @property
    def t(self) -> int:
        """Steps taken (on the GPU: waits for them)."""
        return int(self._steps)

    @t.setter
    def t(self, value: int) -> None:
        self._steps.fill_(int(value))

    def _count(self) -> Tuple[float, float]:
        """One step more; the corrections where the torch form asks."""
        b1, b2 = self.betas
        if self._steps.is_cuda and native_available():
            native().adam_count(self._steps, self._inverse, b1, b2)
            return 1.0, 1.0               # not read: _inverse is
        self._steps.add_(1)
        t = self.t
        return 1 - b1 ** t, 1 - b2 ** t

    def _adamw(self, fp, g, m, v, master, lr, bc1, bc2) -> None:
        b1, b2 = self.betas
        if fp.is_cuda and native_available():
            native().adamw_flat_counted(fp, g, m, v, master, lr, b1, b2,
                                        self.eps, self.weight_decay,
                                        self._inverse)
            return
        g32 = g.float()
        m.mul_(b1).add_(g32, alpha=1 - b1)
        v.mul_(b2).addcmul_(g32, g32, value=1 - b2)
        p32 = master if master is not None else fp.float()
        p32 = p32 - lr * self.weight_decay * p32
        p32 = p32 - lr * (m / bc1) / ((v / bc2).sqrt() + self.eps)
        if master is not None:
            master.copy_(p32)
        fp.copy_(p32.to(fp.dtype))


class FlatAdam(_FlatAdamBase):
    """AdamW over flat buckets (BERT path; fused adamw_flat on HIP)."""

    def __init__(self, engine: DataParallel, lr: float = 1e-4,
                 betas=(0.9, 0.999), eps: float = 1e-8,
                 weight_decay: float = 0.01):
        super().__init__(engine)
        self.lr, self.betas, self.eps = lr, betas, eps
        self.weight_decay = weight_decay
        self.m = [torch.zeros(fp.numel(), dtype=torch.float32,
                              device=fp.device) for fp in self.flat_params]
        self.v = [torch.zeros_like(mm) for mm in self.m]

    @torch.no_grad()
    def step(self) -> None:
        bc1, bc2 = self._count()
        for fp, b, m, v, master in zip(self.flat_params, self.buckets,
                                       self.m, self.v, self.masters):
            self._adamw(fp, b.flat, m, v, master, self.lr, bc1, bc2)

    def state_dict(self) -> dict:
        return {"m": self.m, "v": self.v, "masters": self.masters,
                "t": self.t, "lr": self.lr, "betas": self.betas,
                "eps": self.eps, "weight_decay": self.weight_decay}

    def load_state_dict(self, sd: dict) -> None:
        for dst, src in zip(self.m, sd["m"]):
            dst.copy_(src.to(dst.device))
        for dst, src in zip(self.v, sd["v"]):
            dst.copy_(src.to(dst.device))
        for dst, src in zip(self.masters, sd.get("masters", [])):
            if dst is not None and src is not None:
                dst.copy_(src.to(dst.device))
        self.t = sd["t"]
        self.lr = sd["lr"]
        self.betas = tuple(sd.get("betas", self.betas))
        self.eps = sd.get("eps", self.eps)
        self.weight_decay = sd.get("weight_decay", self.weight_decay)


class FlatMuon(_FlatAdamBase):
    """Muon for hidden matrices, AdamW for the other parameters.

    A hidden matrix is the weight of an ``nn.Linear`` with at least 16 rows
    and columns.  Its step is ``lr * max(1, rows / cols) ** 0.5`` times the
    orthogonalised momentum (``F_amd.newton_schulz``); matrices of one shape
    go through it together.  Embeddings, norms, biases and small heads take
    an AdamW step of ``adam_lr``.  Weight decay is decoupled in both.

    Every rank orthogonalises every matrix from the same averaged gradients,
    bit for bit, so ranks stay in step without an exchange.
    """

    MIN_SIDE = 16

    def __init__(self, engine: DataParallel, lr: float = 0.02,
                 momentum: float = 0.95, nesterov: bool = True,
                 ns_steps: int = 5, ns_eps: float = 1e-7,
                 weight_decay: float = 0.01, adam_lr: float = 3e-4,
                 betas=(0.9, 0.999), eps: float = 1e-8):
        super().__init__(engine)
        self.lr, self.momentum, self.nesterov = lr, momentum, nesterov
        self.ns_steps, self.ns_eps = ns_steps, ns_eps
        self.weight_decay = weight_decay
        self.adam_lr, self.betas, self.eps = adam_lr, betas, eps
        hidden = {id(m.weight) for m in engine.module.modules()
                  if isinstance(m, torch.nn.Linear)
                  and min(m.weight.shape) >= self.MIN_SIDE}
        # a weight that an embedding shares (a tied head) is not hidden
        hidden -= {id(m.weight) for m in engine.module.modules()
                   if isinstance(m, torch.nn.Embedding)}
        # momentum of a matrix, or first moment of anything else
        self.m = [torch.zeros(fp.numel(), dtype=torch.float32,
                              device=fp.device) for fp in self.flat_params]
        # (bucket, start, end) of each matrix, by shape and type ..
        self.groups: Dict[tuple, List[Tuple[int, int, int]]] = {}
        # .. and of each stretch of the rest, with its second moments
        self.rest: List[Tuple[int, int, int]] = []
        for bi, b in enumerate(self.buckets):
            off = 0
            for p in b.params:
                end = off + p.numel()
                if id(p) in hidden:
                    self.groups.setdefault(
                        (*p.shape, p.dtype, p.device), []).append(
                            (bi, off, end))
                elif self.rest and self.rest[-1][0] == bi \
                        and self.rest[-1][2] == off:
                    self.rest[-1] = (bi, self.rest[-1][1], end)
                else:
                    self.rest.append((bi, off, end))
                off = end
        # the fused AdamW takes four elements at a time from where a stretch
        # begins: up to three in front of such a border are one of their own
        self.rest = [span for bi, a, e in self.rest
                     for span in ((bi, a, min(e, -(-a // 4) * 4)),
                                  (bi, min(e, -(-a // 4) * 4), e))
                     if span[1] < span[2]]
        self.v = [torch.zeros(e - a, dtype=torch.float32,
                              device=self.flat_params[bi].device)
                  for bi, a, e in self.rest]

    def _matrices(self, spans):
        cut = lambda flats: [flats[bi][a:e] for bi, a, e in spans]  # noqa: E731
        masters = [] if self.masters[spans[0][0]] is None \
            else cut(self.masters)
        return (cut(self.flat_params), cut([b.flat for b in self.buckets]),
                cut(self.m), masters)

    def _step_matrices(self, rows: int, cols: int, spans) -> None:
        params, grads, moms, masters = self._matrices(spans)
        step = self.lr * max(1.0, rows / cols) ** 0.5
        keep = 1.0 - self.lr * self.weight_decay
        u = torch.empty(len(spans), rows, cols, dtype=torch.float32,
                        device=params[0].device)
        if u.is_cuda and native_available():
            native().muon_momentum(grads, moms, u, self.momentum,
                                   self.nesterov)
            o = F_amd.newton_schulz(u, self.ns_steps, self.ns_eps)
            native().muon_apply(params, masters, o, step, keep)
            return
        for i, (g, m) in enumerate(zip(grads, moms)):
            m.mul_(self.momentum).add_(g.float())
            u[i] = (g.float().add(m, alpha=self.momentum) if self.nesterov
                    else m).view(rows, cols)
        o = F_amd.newton_schulz(u, self.ns_steps, self.ns_eps).float()
        for i, p in enumerate(params):
            w = masters[i] if masters else p
            w.copy_(keep * w.float() - step * o[i].reshape(-1))
            if masters:
                p.copy_(w.to(p.dtype))

    def _step_rest(self, span, v: torch.Tensor, bc1: float,
                   bc2: float) -> None:
        bi, a, e = span
        master = self.masters[bi]
        self._adamw(self.flat_params[bi][a:e], self.buckets[bi].flat[a:e],
                    self.m[bi][a:e], v,
                    None if master is None else master[a:e], self.adam_lr,
                    bc1, bc2)

    @torch.no_grad()
    def step(self) -> None:
        bc1, bc2 = self._count()
        for (rows, cols, _, _), spans in self.groups.items():
            self._step_matrices(rows, cols, spans)
        for span, v in zip(self.rest, self.v):
            self._step_rest(span, v, bc1, bc2)

    def state_dict(self) -> dict:
        return {"m": self.m, "v": self.v, "masters": self.masters,
                "t": self.t, "lr": self.lr, "momentum": self.momentum,
                "nesterov": self.nesterov, "ns_steps": self.ns_steps,
                "ns_eps": self.ns_eps, "adam_lr": self.adam_lr,
                "betas": self.betas, "eps": self.eps,
                "weight_decay": self.weight_decay}

    def load_state_dict(self, sd: dict) -> None:
        for mine, theirs in ((self.m, sd["m"]), (self.v, sd["v"]),
                             (self.masters, sd.get("masters", []))):
            for dst, src in zip(mine, theirs):
                if dst is not None and src is not None:
                    dst.copy_(src.to(dst.device))
        for k in ("t", "lr", "momentum", "nesterov", "ns_steps", "ns_eps",
                  "adam_lr", "eps", "weight_decay"):
            setattr(self, k, sd[k])
        self.betas = tuple(sd["betas"])
