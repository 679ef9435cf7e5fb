"""Gradient descent with momentum on an iPEPS (reference optim/ad_optim_sgd_mod.py): `optimize_state` with the interface, the log, the
checkpoints and the stopping rules of ad_optim_lbfgs_mod.optimize_state, OPTARGS.lr / momentum / dampening, and a bound on the norm of the
gradient, OPTARGS.clip_grad_norm.  The update of all on-site tensors, the scaling included, is one call of the native engine
(optim.grads.sgd_step)."""
import torch
import config as cfg
from optim import ad_optim_lbfgs_mod, grads


class SGD(torch.optim.Optimizer):
    """torch.optim.SGD's iteration (lr, momentum, dampening) with the gradient scaled to 2-norm (or largest modulus, norm_type inf) at most `max_norm`
    over all parameters; `.grad` is not changed.  `norms` of the last step: device tensor [2-norm, largest modulus] of the raw gradient, None
    without `max_norm`.  One parameter group, of one dtype on the engine's device, whose lr, momentum, dampening and max_norm may be changed between
    steps; a graph that captured a step keeps those of the capture, and is captured after the first step (which makes the momentum buffers).  A step
    that raises leaves parameters and buffers as they were."""

    norms = None

    def __init__(self, params, lr, momentum=0.0, dampening=0.0, max_norm=None, norm_type=2):
        for k, v in (("lr", lr), ("momentum", momentum), ("max_norm", 0.0 if max_norm is None else max_norm)):
            if not v >= 0.0:
                raise ValueError(f"invalid {k}: {v}")
        if norm_type not in (2, float("inf")):
            raise ValueError(f"invalid norm_type: {norm_type}")
        super().__init__(params, dict(lr=lr, momentum=momentum, dampening=dampening, max_norm=max_norm, norm_type=norm_type))
        if len(self.param_groups) != 1:
            raise ValueError("SGD: one parameter group only (the norm is that of all parameters)")

    def load_state_dict(self, state_dict):
        """Of this class or of torch.optim.SGD, which has no bound; what it has besides (weight_decay, nesterov, maximize) is refused."""
        groups = []
        for g in state_dict["param_groups"]:
            for k in ("weight_decay", "nesterov", "maximize"):
                if g.get(k):
                    raise ValueError(f"SGD: {k} {g[k]} of the stored state")
            groups.append({"max_norm": None, "norm_type": 2, **g})
        super().load_state_dict({**state_dict, "param_groups": groups})

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        group = self.param_groups[0]
        ps = [p for p in group["params"] if p.grad is not None]
        gs = [p.grad for p in ps]
        kw = dict(lr=group["lr"], momentum=group["momentum"], dampening=group["dampening"])
        bound = dict(max_norm=group["max_norm"], norm_type=group["norm_type"])
        if group["momentum"] == 0.0:
            self.norms = grads.sgd_step(ps, gs, **kw, **bound)
            return loss
        # (a call that fails leaves no trace: new buffers count from the call on that has filled them)
        bufs = [self.state.get(p, {}).get("momentum_buffer") for p in ps]
        new = [i for i, m in enumerate(bufs) if m is None]
        for i in new:
            bufs[i] = torch.empty_like(ps[i])
        if len(new) in (0, len(ps)):
            norms = grads.sgd_step(ps, gs, bufs, first=len(new) > 0, **kw, **bound)
        else:
            # some parameters take their first step, the others do not: two calls, the factor is that of all gradients
            norms = None
            if bound["max_norm"] is not None:
                scaled = [torch.empty_like(g) for g in gs]
                norms = grads.clip_grads(gs, out=scaled, **bound)
                gs = scaled
            before = [ps[i].clone() for i in new]
            grads.sgd_step([ps[i] for i in new], [gs[i] for i in new], [bufs[i] for i in new], first=True, **kw)
            rest = [i for i in range(len(ps)) if i not in new]
            try:
                grads.sgd_step([ps[i] for i in rest], [gs[i] for i in rest], [bufs[i] for i in rest], **kw)
            except BaseException:
                for i, x in zip(new, before):
                    ps[i].copy_(x)
                raise
        for i in new:
            self.state[ps[i]]["momentum_buffer"] = bufs[i]
        self.norms = norms
        return loss


def create_optimizer(state, main_args=cfg.main_args, opt_args=cfg.opt_args, ctm_args=cfg.ctm_args, global_args=cfg.global_args):
    parameters = list(state.get_parameters())
    for A in parameters:
        A.requires_grad_(True)
    if opt_args.line_search not in (None, "default"):
        raise RuntimeError("unsupported line search")
    optimizer = SGD(parameters, lr=opt_args.lr, momentum=opt_args.momentum, dampening=opt_args.dampening,
                    max_norm=opt_args.clip_grad_norm if opt_args.clip_grad_norm > 0.0 else None)
    optimizer.zero_grad()
    return parameters, optimizer


def load_optimizer_state_(optimizer, state, main_args=cfg.main_args, opt_args=cfg.opt_args, ctm_args=cfg.ctm_args,
                          global_args=cfg.global_args):
    """Resume from `main_args.opt_resume`, a checkpoint of this optimiser or of torch.optim.SGD (whose bound is that of the current OPTARGS); with
    `opt_resume_override_params` the stored lr, momentum, dampening and bound are replaced by the current OPTARGS."""
    print(f"INFO: resuming from check point. resume = {main_args.opt_resume}")
    checkpoint = torch.load(main_args.opt_resume, map_location=state.device, weights_only=False)
    sd = checkpoint["optimizer_state_dict"]
    group = sd["param_groups"][0]
    if "dampening" not in group:
        raise RuntimeError(f"{main_args.opt_resume} is not a checkpoint of gradient descent")
    group.setdefault("max_norm", optimizer.param_groups[0]["max_norm"])          # (a checkpoint of torch.optim.SGD)
    if main_args.opt_resume_override_params:
        group.update(lr=opt_args.lr, momentum=opt_args.momentum, dampening=opt_args.dampening,
                     max_norm=opt_args.clip_grad_norm if opt_args.clip_grad_norm > 0.0 else None)
    optimizer.load_state_dict(sd)
    print(f"checkpoint.loss = {checkpoint['loss']}")


def optimize_state(state, ctm_env_init, loss_fn, obs_fn=None, post_proc=None, main_args=cfg.main_args, opt_args=cfg.opt_args,
                   ctm_args=cfg.ctm_args, global_args=cfg.global_args):
    """ad_optim_lbfgs_mod.optimize_state with gradient descent in the place of L-BFGS: one evaluation and one step per epoch."""
    ad_optim_lbfgs_mod.optimize_state(state, ctm_env_init, loss_fn, obs_fn=obs_fn, post_proc=post_proc, main_args=main_args, opt_args=opt_args,
                                      ctm_args=ctm_args, global_args=global_args, create=create_optimizer, load=load_optimizer_state_)
