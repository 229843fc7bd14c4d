"""A token-mixer block over latent planes, built from lama_b200.operators (no counterpart in the
reference): an alternative to a spectral block's global branch that takes a plane as a raster of
tokens, in linear time, and can take it in strips or token by token with a carried state.

A block maps the residual stream u and its norm n to the next ones:

    y = W_o linear_attention(W_q n, W_k n, W_v n)
    u', n' = gated_residual_norm(u, y)      # norm of y, gate, residual scale, sum, norm for the next block

`forward` runs whole sequences, in training with the norms' activations kept in 8 bits; `step` runs one
token a stream.  `python -m lama_b200.mixer` (with this package's directory on the path) trains a small
stack for a few steps and streams through it.
"""

from __future__ import annotations

import math

import torch

from . import operators as F


class TokenMixer(torch.nn.Module):
    """One block: `heads` heads of `dk` and `dv` channels over a stream of `channels`, fixed decays from a
    memory of about one token to about `memory` tokens."""

    def __init__(self, channels=512, heads=8, dk=64, dv=64, memory=4096.0, save="int8", device="cuda",
                 dtype=torch.bfloat16):
        super().__init__()
        if save not in ("full", "int8"):
            raise ValueError("save is 'full' or 'int8'")
        self.heads, self.dk, self.dv, self.save = heads, dk, dv, save
        kw = dict(device=device, dtype=dtype)
        self.qkv = torch.nn.Linear(channels, heads * (2 * dk + dv), bias=False, **kw)
        self.out = torch.nn.Linear(heads * dv, channels, bias=False, **kw)
        self.post_weight = torch.nn.Parameter(torch.ones(channels, device=device))
        self.pre_weight = torch.nn.Parameter(torch.ones(channels, device=device))
        self.residual_scale = torch.nn.Parameter(torch.full((channels,), 0.1, device=device))
        i = torch.arange(heads, device=device, dtype=torch.float32) / max(heads - 1, 1)
        self.register_buffer("log_decay", -torch.exp(-i * math.log(memory)))

    def _project(self, n):
        """q, k, v as views of one projection (the operators take their strides)."""
        h, dk, dv = self.heads, self.dk, self.dv
        x = self.qkv(n)
        q, k, v = x.split((h * dk, h * dk, h * dv), -1)
        return q.unflatten(-1, (h, dk)), k.unflatten(-1, (h, dk)), v.unflatten(-1, (h, dv))

    def _close(self, u, y, gate):
        return F.gated_residual_norm(u, y, post_weight=self.post_weight, pre_weight=self.pre_weight, gate=gate,
                                     residual_scale=self.residual_scale, save=self.save if self.training else None)[:2]

    def forward(self, u, n, gate=None, state=None, lengths=None):
        """u, n: [B,T,C]; gate: None, [B,1,C] or [B,T,C]; state: of the tokens before, or None.
        Returns (u', n', state after the last token)."""
        q, k, v = self._project(n)
        o, state = F.linear_attention(q, k, v, self.log_decay, initial_state=state, lengths=lengths, return_state=True)
        return *self._close(u, self.out(o.flatten(-2)), gate), state

    @torch.no_grad()
    def step(self, u, n, state, gate=None, slots=None):
        """One token a row: u, n [B,C], gate None or [B,C]; state [N,H,dk,dv], updated in place.  Returns (u', n')."""
        q, k, v = self._project(n)
        o = F.linear_attention_step(q, k, v, self.log_decay, state, slots=slots)
        u, n = F.gated_residual_norm(u, self.out(o.flatten(-2)), post_weight=self.post_weight,
                                     pre_weight=self.pre_weight, gate=gate, residual_scale=self.residual_scale)
        return u, n

    def new_state(self, rows):
        return torch.zeros(rows, self.heads, self.dk, self.dv, device=self.log_decay.device)


def main(steps=60, side=32, channels=128, blocks=2):
    """Fills the hidden half of a few smooth planes: trains a small stack, then streams it token by token."""
    torch.manual_seed(0)
    stack = torch.nn.ModuleList(TokenMixer(channels, heads=2, memory=side * side) for _ in range(blocks))
    opt = torch.optim.Adam(stack.parameters(), 3e-3)
    yy, xx = torch.meshgrid(*(torch.linspace(0, 6.28, side, device="cuda"),) * 2, indexing="ij")
    losses = []
    token = 0.3 * torch.randn(channels, device="cuda")  # stands in hidden places: a query of zeros would read nothing
    f = torch.rand(4, channels, 2, 1, 1, device="cuda") * 2
    plane = torch.sin(f[:, :, 0] * yy + f[:, :, 1] * xx).flatten(2).transpose(1, 2)  # [B, side*side, C]
    for _ in range(steps):
        hidden = (torch.rand(4, side * side, 1, device="cuda") < 0.5).float()
        u = n = (plane * (1 - hidden) + token * hidden).bfloat16()
        for block in stack:
            u, n, _ = block(u, n)
        loss = ((u.float() - plane).square() * hidden).mean()
        opt.zero_grad()
        loss.backward()
        opt.step()
        losses.append(float(loss.detach()))
    print(f"loss {losses[0]:.4f} -> {losses[-1]:.4f} over {steps} steps")
    stack.eval()
    with torch.no_grad():
        u = n = x = (plane * (1 - hidden) + token * hidden).bfloat16()
        for block in stack:
            u, n, _ = block(u, n)
        states = [block.new_state(4) for block in stack]
        worst = 0.0
        for t in range(64):
            a = b = x[:, t]
            for block, s in zip(stack, states):
                a, b = block.step(a, b, s)
            worst = max(worst, float((a.float() - u[:, t].float()).abs().max()))
    F.check_operators()
    print(f"64 streamed tokens: within {worst:.3g} of the whole-sequence pass")
    return losses, worst


if __name__ == "__main__":
    main()
