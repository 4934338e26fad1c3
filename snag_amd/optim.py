"""Optimiser / schedule construction around the model, as the reference's training loop does it (src/utils.py:25-86 ``set_optim``,
called from main.py:92): parameter groups by NAME -- for ``model_name == "SNAG"`` anything containing ``weight_raw`` / ``bias`` /
``multi_loss_layer`` is not decayed and ``multi_loss_layer`` runs at 5x the learning rate -- AdamW or Adam, and the fixed / linear /
cosine schedules with warm-up.  Plain host code on torch.optim: the drop-in ``snag_amd.mmea.SNAG`` keeps the reference's parameter
names, so the groups come out identical (golden G14).

Not in the reference: ``orthogonalize`` / ``muon_step`` (HIP, csrc/muon.hip) and the ``Muon`` optimiser, which ``set_optim`` builds for
``opt.optim == "muon"`` -- each group above is then cut into its matrices (Muon, at ``opt.muon_lr``, without it at the group's own AdamW rate) and the
rest (AdamW); Muon's momentum, steps and scaling keep their defaults there."""
import torch
from torch import optim
from torch.optim.adamw import adamw

from . import ops


def orthogonalize(matrices, steps=5, eps=1e-7):
    """Newton-Schulz orthogonalisation on the matrix pipe: X = G / (|G|_F + eps), then ``steps`` times X <- a X + (b A + c A^2) X with
    A = X X^T and (a, b, c) = (3.4445, -4.7750, 2.0315), which takes every singular value that is not tiny into about 0.7 .. 1.2.
    One matrix or a list of matrices of one type (fp32, bf16, fp16) -> the same, new tensors, detached: not differentiable.  All matrices of a list share the
    launches.  Products take operands of 22 bits for fp32 and fp16 matrices, of 11 off the diagonal for bf16 (5e-4 where the result's rounding is 1.7e-3)."""
    if torch.is_tensor(matrices):
        return ops.orthogonalize([matrices.detach()], steps=steps, eps=eps)[0]
    return ops.orthogonalize([m.detach() for m in matrices], steps=steps, eps=eps)


def muon_step(weights, grads, momenta, lr, momentum=0.95, nesterov=True, weight_decay=0.0, match_rms=False, steps=5, eps=1e-7):
    """One Muon update of a list of matrices, in place: M <- mu M + (1 - mu) G; U = (1 - mu) G + mu M (``nesterov``) or M;
    W <- (1 - lr weight_decay) W - lr s orthogonalize(U), s = sqrt(max(1, rows / cols)) or, with ``match_rms``, 0.2 sqrt(max(rows, cols)).
    ``momenta`` are fp32, ``grads`` of the weights' type; U enters the products as orthogonalize's matrices of that type do."""
    ops.muon_step([w.detach() for w in weights], [g.detach() for g in grads], momenta, lr, momentum, nesterov, weight_decay, match_rms, steps, eps)


class Muon(optim.Optimizer):
    """Muon for matrices (``muon=True`` groups, the default: every parameter is 2-D) and AdamW for what is none (``muon=False`` groups), as one
    torch optimiser.  State: fp32 ``momentum_buffer`` per matrix."""

    def __init__(self, params, lr=0.02, momentum=0.95, nesterov=True, weight_decay=0.0, match_rms=False, steps=5, eps=1e-7, betas=(0.9, 0.999), adam_eps=1e-8):
        if lr < 0 or weight_decay < 0 or not 0 <= momentum < 1:
            raise ValueError(f"Muon: lr {lr}, momentum {momentum}, weight_decay {weight_decay}")
        super().__init__(params, dict(lr=lr, momentum=momentum, nesterov=nesterov, weight_decay=weight_decay, match_rms=match_rms, steps=steps, eps=eps,
                                      betas=betas, adam_eps=adam_eps, muon=True))

    def add_param_group(self, group):
        super().add_param_group(group)
        group = self.param_groups[-1]
        if group["muon"] and any(p.dim() != 2 for p in group["params"]):
            self.param_groups.pop()
            raise ValueError("Muon: a parameter that is not a matrix (put it into a group with muon=False)")

    def load_state_dict(self, state_dict):
        """torch casts the state to its parameter's type: the momentum of a 16-bit matrix is put back as it was saved, in fp32."""
        super().load_state_dict(state_dict)
        saved = (i for g in state_dict["param_groups"] for i in g["params"])
        for i, p in zip(saved, (p for g in self.param_groups for p in g["params"])):
            m = state_dict["state"].get(i, {}).get("momentum_buffer")
            if m is not None:
                self.state[p]["momentum_buffer"] = m.to(device=p.device, dtype=torch.float32).contiguous()

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            ps = [p for p in group["params"] if p.grad is not None]
            if group["muon"]:
                self._muon(group, ps)
            elif ps:
                self._adamw(group, ps)
        return loss

    def _muon(self, group, ps):
        for p in ps:
            if not self.state[p]:
                self.state[p]["momentum_buffer"] = torch.zeros_like(p, dtype=torch.float32, memory_format=torch.contiguous_format)
        lists = {}                                       # one call per type and device
        for p in ps:
            lists.setdefault((p.dtype, p.device), []).append(p)
        for same in lists.values():
            muon_step(same, [p.grad.contiguous() for p in same], [self.state[p]["momentum_buffer"] for p in same], group["lr"], group["momentum"],
                      group["nesterov"], group["weight_decay"], group["match_rms"], group["steps"], group["eps"])

    def _adamw(self, group, ps):
        for p in ps:
            st = self.state[p]
            if not st:
                st["step"], st["exp_avg"], st["exp_avg_sq"] = torch.zeros(()), torch.zeros_like(p), torch.zeros_like(p)
        st = [self.state[p] for p in ps]
        adamw(ps, [p.grad for p in ps], [s["exp_avg"] for s in st], [s["exp_avg_sq"] for s in st], [], [s["step"] for s in st], amsgrad=False,
              beta1=group["betas"][0], beta2=group["betas"][1], lr=group["lr"], weight_decay=group["weight_decay"], eps=group["adam_eps"], maximize=False)


def _is_matrix(name, p):
    """What Muon updates: matrices that are multiplied by; tables that rows are looked up in and weights of other ranks stay with AdamW."""
    return p.dim() == 2 and min(p.shape) > 1 and max(p.shape) <= ops.MUON_MAX_SIDE and "emb" not in name


def set_optim(opt, model_list, freeze_part=(), no_freeze_part=(), accumulation_step=None):
    """-> (optimizer, scheduler).  ``opt`` carries model_name, lr, weight_decay, adam_epsilon, optim, scheduler, warmup_steps,
    total_steps, accumulation_steps -- the fields the reference reads."""
    named = []
    for model in model_list:
        for n, p in model.named_parameters():
            trainable = not any(nd in n for nd in freeze_part) and (len(no_freeze_part) == 0 or any(nd in n for nd in no_freeze_part))
            if trainable:
                named.append((n, p))
            else:
                p.requires_grad = False
    if opt.model_name == "SNAG":
        no_decay, large_lr = ["weight_raw", "bias", "multi_loss_layer"], ["multi_loss_layer"]
        plain = lambda n: any(nd in n for nd in no_decay)
        large = lambda n: any(nd in n for nd in large_lr)
        groups = [
            {"params": [p for n, p in named if not plain(n)], "lr": opt.lr, "weight_decay": opt.weight_decay},
            {"params": [p for n, p in named if plain(n) and not large(n)], "lr": opt.lr, "weight_decay": 0.0},
            {"params": [p for n, p in named if plain(n) and large(n)], "lr": 5 * opt.lr, "weight_decay": 0.0},
        ]
    else:
        groups = [{"params": [p for _, p in named], "lr": opt.lr, "weight_decay": opt.weight_decay}]
    if opt.optim == "adamw":
        optimizer = optim.AdamW(groups, lr=opt.lr, eps=opt.adam_epsilon)
    elif opt.optim == "adam":
        optimizer = optim.Adam(groups, lr=opt.lr)
    elif opt.optim == "muon":
        names = {p: n for n, p in named}
        cut = []
        for g in groups:
            for muon in (True, False):
                ps = [p for p in g["params"] if _is_matrix(names[p], p) == muon]
                if ps:
                    cut.append({**g, "params": ps, "muon": muon, "lr": getattr(opt, "muon_lr", g["lr"]) if muon else g["lr"]})
        optimizer = Muon(cut, lr=opt.lr, adam_eps=opt.adam_epsilon)
    else:
        raise ValueError(f"unknown optimiser {opt.optim!r}")
    if accumulation_step is None:
        accumulation_step = opt.accumulation_steps
    if opt.scheduler == "fixed":
        scheduler = torch.optim.lr_scheduler.LambdaLR(optimizer, lambda step: 1.0)
    elif opt.scheduler in ("linear", "cos"):
        from transformers import get_cosine_schedule_with_warmup, get_linear_schedule_with_warmup
        make = get_linear_schedule_with_warmup if opt.scheduler == "linear" else get_cosine_schedule_with_warmup
        scheduler = make(optimizer, num_warmup_steps=int(opt.warmup_steps / accumulation_step),
                         num_training_steps=int(opt.total_steps / accumulation_step))
    else:
        raise ValueError(f"unknown scheduler {opt.scheduler!r}")
    return optimizer, scheduler
