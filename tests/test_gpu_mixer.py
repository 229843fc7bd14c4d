"""The token-mixer block (lama_b200.mixer) as it is used: a training step against a plain fp64 block, strips and
single tokens against the whole sequence, and the packaged example."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def plain_block(m, u, n, gate):
    """The block in 64 bits from the formulas alone."""
    h, dk, dv = m.heads, m.dk, m.dv
    B, T, _ = u.shape
    x = n @ m.qkv.weight.T
    q, k, v = (p.view(B, T, h, -1).transpose(1, 2) for p in x.split((h * dk, h * dk, h * dv), -1))
    pos = torch.arange(T, device=u.device, dtype=torch.float64)
    d = pos[:, None] - pos[None]
    decay = torch.where(d >= 0, torch.exp(m.log_decay.double()[:, None, None] * d.clamp_min(0)), 0.0)
    o = ((q @ k.transpose(-1, -2)) * decay * dk ** -0.5) @ v
    y = o.transpose(1, 2).reshape(B, T, h * dv) @ m.out.weight.T
    norm = lambda t: t / torch.sqrt((t * t).mean(-1, keepdim=True) + 1e-6)  # noqa: E731
    u = u + m.residual_scale * gate * m.post_weight * norm(y)
    return u, m.pre_weight * norm(u)


def test_training_step_matches_a_plain_block():
    """fp32 end to end: the products of the projections are torch's own, so the bound is that of fp32 sums of
    about 500 terms in each of five stages, 1e-4 of each result's size, and wide of that for any wrong term."""
    from lama_b200.mixer import TokenMixer
    torch.manual_seed(1)
    m = TokenMixer(96, heads=2, dk=32, dv=48, memory=200.0, save="full", dtype=torch.float32)
    u = torch.randn(2, 300, 96, device="cuda", requires_grad=True)
    n = torch.randn(2, 300, 96, device="cuda", requires_grad=True)
    gate = torch.randn(2, 1, 96, device="cuda", requires_grad=True)
    a, b, _ = m(u, n, gate)
    wa, wb = torch.randn_like(a), torch.randn_like(b)
    ((a * wa).sum() + (b * wb).sum()).backward()
    got = {k: p.grad.clone() for k, p in m.named_parameters()} | {"u": u.grad, "n": n.grad, "gate": gate.grad}
    m64 = TokenMixer(96, heads=2, dk=32, dv=48, memory=200.0, save="full", dtype=torch.float32)
    m64.load_state_dict(m.state_dict())
    m64 = m64.double()
    ins = [t.detach().double().requires_grad_() for t in (u, n, gate)]
    ea, eb = plain_block(m64, *ins)
    ((ea * wa).sum() + (eb * wb).sum()).backward()
    exp = {k: p.grad for k, p in m64.named_parameters()} | dict(zip(("u", "n", "gate"), (t.grad for t in ins)))
    for x, y in ((a, ea), (b, eb)):
        assert (x.double() - y).norm() <= 1e-4 * y.norm()
    assert got.keys() == exp.keys()
    for k in got:
        assert (got[k].double() - exp[k]).norm() <= 1e-4 * exp[k].norm(), k


def test_int8_checkpoints_change_gradients_by_their_rounding_alone():
    """Codes hold 1/254 of a group's largest value; for normal activations that is about 1 % of a value's size, and
    the gradients pass through one or two of them."""
    from lama_b200.mixer import TokenMixer
    grads = {}
    for save in ("full", "int8"):
        torch.manual_seed(2)
        m = TokenMixer(256, heads=4, save=save, dtype=torch.float32)
        u = torch.randn(2, 200, 256, device="cuda", requires_grad=True)
        a, b, _ = m(u, u)
        (a.square().sum() + (b * torch.arange(256, device="cuda")).sum()).backward()
        grads[save] = u.grad
    off = (grads["int8"] - grads["full"]).norm() / grads["full"].norm()
    assert 0 < off <= 0.03


def test_strips_and_steps_continue_the_sequence():
    """Three strips and single tokens against the whole: both round the same values to bf16 at the same places, the
    sums differ in fp32; a flipped bf16 rounding (2^-8) may spread through one block."""
    from lama_b200.mixer import TokenMixer
    torch.manual_seed(3)
    m = TokenMixer(128, heads=2).eval()
    u = torch.randn(2, 400, 128, device="cuda").bfloat16()
    with torch.no_grad():
        a, b, s = m(u, u)
        state, parts = None, []
        for lo, hi in ((0, 100), (100, 391), (391, 400)):
            x, _, state = m(u[:, lo:hi], u[:, lo:hi], state=state)
            parts.append(x)
        assert (torch.cat(parts, 1).float() - a.float()).norm() <= 2 ** -8 * a.float().norm()
        assert (state - s).norm() <= 1e-4 * s.norm()
        _, _, state = m(u[:, :390], u[:, :390])
        for t in range(390, 400):
            x, _ = m.step(u[:, t], u[:, t], state)
            assert (x.float() - a[:, t].float()).norm() <= 2 ** -6 * a[:, t].float().norm()


def test_the_example_learns_and_streams():
    from lama_b200 import mixer
    losses, worst = mixer.main()
    assert losses[-1] < losses[0]
    assert worst <= 0.1
