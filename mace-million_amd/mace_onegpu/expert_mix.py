"""ExpertMix: a mixture of expert linears on equivariant node features, and a command that fits one on pass A's
features.

Where the species-block skip multiplies an atom's features by the block of its species (SpeciesSkip of the reference,
fast_layers.py:41-105), a mixture gives every atom k of E blocks with learned gates: norm of the scalars, a router,
route, plan_experts, and one expert_linear per l, whose 2 l + 1 components share the atom's experts, so the map stays
equivariant.

    python -m mace_onegpu.expert_mix --water 64 --steps 60

evaluates the structure, takes the layer-1 features H1, and fits a mixture with a linear readout to the atoms' energies
(layer 2's part, standardised), by Adam with a bias that keeps the experts' loads even.

The choice of experts jumps where two of an atom's keys cross.  An energy that has to be smooth in the positions is
routed by something that does not move with the atoms (`by`: species embeddings, say); per-atom properties may be routed
by the features themselves.
"""
import math

import torch

from .experts import expert_linear, plan_experts, route
from .layer_norm import LayerNorm


class ExpertMix(torch.nn.Module):
    """out[i, l, :] = sum_j gates[i, j] h[i, l, :] @ blocks[l][experts[i, j]] for ir_mul features h [N, components, C]
    (or [N, components C]) with irreps ls (every one C channels); gates and experts from the layer norm of `by` [N, C]
    (the scalars of h).  balance [n_experts] is added to the logits for the choice alone; update_balance moves it
    against the loads of the last call."""

    def __init__(self, channels=128, ls=(0, 1), n_experts=8, k=2, scoring="softmax", groups=1, top_groups=None,
                 renormalize=True, seed=0, dtype=torch.float32, device="cuda"):
        super().__init__()
        g = torch.Generator().manual_seed(seed)
        rn = lambda *shape: (torch.randn(*shape, generator=g) / math.sqrt(shape[-2])).to(dtype).to(device)  # noqa: E731
        self.ls, self.k, self.n_experts = tuple(ls), int(k), int(n_experts)
        self.route_args = dict(scoring=scoring, groups=groups, top_groups=top_groups, renormalize=renormalize)
        self.norm = LayerNorm(channels, dtype=dtype, device=device)
        self.router = torch.nn.Parameter(rn(channels, n_experts))
        self.blocks = torch.nn.ParameterList([rn(n_experts, channels, channels) for _ in self.ls])
        self.register_buffer("balance", torch.zeros(n_experts, device=device))
        self.plan = None        # of the last call

    def __getstate__(self):     # copies and saved modules go without it
        return dict(super().__getstate__(), plan=None)

    def forward(self, h, by=None):
        n_comp = sum(2 * l + 1 for l in self.ls)
        C = self.blocks[0].shape[1]
        if h.dim() == 2:
            h = h.view(h.shape[0], -1, C)
        if h.dim() != 3 or h.shape[1:] != (n_comp, C):
            raise ValueError(f"features must be [atoms, {n_comp}, {C}] or [atoms, {n_comp * C}], got {tuple(h.shape)}")
        logits = self.norm(h[:, 0] if by is None else by) @ self.router
        gates, experts = route(logits, self.k, bias=self.balance, **self.route_args)
        self.plan = plan_experts(experts, self.n_experts)
        out, at = [], 0
        for l, block in zip(self.ls, self.blocks):
            out.append(expert_linear(h[:, at:at + 2 * l + 1], block, self.plan, gates))
            at += 2 * l + 1
        return torch.cat(out, 1)

    @torch.no_grad()
    def update_balance(self, rate=1e-2):
        """Lowers the keys of the experts that had more than the mean load in the last call, raises the others'."""
        load = self.plan.counts.float()
        self.balance -= rate * torch.sign(load - load.mean())


def main(argv=None):
    """Fit a mixture of expert linears with a linear readout to the atoms' energies on the layer-1 features."""
    import argparse

    import numpy as np

    from . import systems
    from .model import from_arg
    from .receiver_chunk_mace import ReceiverChunkMACE, System

    ap = argparse.ArgumentParser(prog="python -m mace_onegpu.expert_mix", description=main.__doc__)
    ap.add_argument("--model", default="seed:0", help='"seed:N" (random-init weights) or a weights file')
    systems.add_structure_args(ap)
    ap.add_argument("--chunk", type=int, default=131072, help="receivers per chunk of the evaluation")
    ap.add_argument("--experts", type=int, default=8)
    ap.add_argument("--k", type=int, default=2, help="experts per atom")
    ap.add_argument("--steps", type=int, default=60)
    ap.add_argument("--lr", type=float, default=3e-3)
    a = ap.parse_args(argv)
    if not torch.cuda.is_available():
        raise SystemExit("the operators run on the GPU; no GPU is visible")
    model = from_arg(a.model)
    pos, box, Z, _ = systems.structure_from_args(a)
    s = System(pos, box, np.asarray(Z) - 1, float(model.spec.r_max), "cuda")
    s.build_neighbors()
    ev = ReceiverChunkMACE(model, chunk=a.chunk, device="cuda")
    _, eat, _, _ = ev.compute(s)
    h = ev.H1.view(s.N, 4, -1)
    h = h / h.square().mean().sqrt()
    target = ((eat - eat.mean()) / eat.std()).float()
    mix = ExpertMix(channels=h.shape[2], n_experts=a.experts, k=a.k)
    readout = torch.nn.Linear(h.shape[2], 1, device="cuda")
    opt = torch.optim.Adam([*mix.parameters(), *readout.parameters()], lr=a.lr)
    losses = []
    for step in range(a.steps):
        out = mix(h)
        # the scalars, and the invariant that the vectors give (their squares, channel by channel)
        loss = (readout(torch.nn.functional.silu(out[:, 0]) + out[:, 1:].square().sum(1)).squeeze(1)
                - target).square().mean()
        opt.zero_grad()
        loss.backward()
        opt.step()
        mix.update_balance()
        losses.append(float(loss.detach()))
        if step % 10 == 0 or step + 1 == a.steps:
            print(f"step {step}: loss {losses[-1]:.4f}  load {mix.plan.counts.tolist()}", flush=True)
    with torch.no_grad():                     # one atom alone, as a trial move needs it, against all atoms at once
        diff = float((mix(h[:1]) - mix(h)[:1]).abs().max())
    print(f"one atom alone differs from the whole box by {diff:.2e}", flush=True)
    return dict(losses=losses, single=diff, atoms=s.N)


if __name__ == "__main__":
    main()
