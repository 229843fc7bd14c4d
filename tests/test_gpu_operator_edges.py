"""The token-mixer operators where their inner number formats could give way: weight that lies far back
in a fast-decaying sequence, long sequences, many gate rows; and what a caller's autograd sees of them.

The bounds are those of test_gpu_operators.py.  For fp16 they hold at the lower end too, up to what the scales
in front of the roundings lose: a score is kept to 2^-38 of its row's largest (decayed, unmasked) one and a decayed
operand to 2^-39 of its chunk's largest, both far below the fp32 sums' share of the bound where the other
factor's sizes do not spread as far.  Where that factor is zero for the largest ones (few tokens with a gradient under dense
queries) the loss itself is the bound.  2^-25 is half of fp16's smallest number.
"""

import pytest
import torch

from test_gpu_operators import (F, UNIT, attention64, bound, close, decays, gen, norm64, norm_inputs, randn,  # noqa: F401
                                state_bound)

pytestmark = pytest.mark.gpu

HALF_FLOOR = 2.0 ** -25


def sparse(x, tokens):
    """x with nothing but the given tokens of each run of 128 left."""
    keep = torch.zeros(x.shape[1], dtype=torch.bool, device="cuda")
    for t in tokens:
        keep[t::128] = True
    return x * keep[None, :, None, None]


FAR = [(250, 64, 64, 2), (700, 64, 128, 2), (2500, 128, 64, 1), (300, 128, 128, 2)]


@pytest.mark.parametrize("T,dk,dv,hv", FAR)
def test_fp16_weight_that_lies_far_back(F, T, dk, dv, hv):  # noqa: F811
    """Large queries and keys, most keys zero, a decay that halves each token: what a row still sees of a key
    30 to 60 tokens back is far below the products' size, and well inside fp16 as a result."""
    g = gen(71)
    q, k = (randn(g, 2, T, 2, dk) * 200).half(), (randn(g, 2, T, 2, dk) * 200).half()
    v = (randn(g, 2, T, hv, dv) * 0.1).half()
    k = sparse(k, (1, 84))
    ld, scale = torch.tensor([-0.7, -0.05], device="cuda"), 0.125
    o, s = F.linear_attention(q, k, v, ld, scale=scale, return_state=True)
    eo, es = attention64(q, k, v, ld, scale)
    mo, ms = attention64(q, k, v, ld, scale, absolute=True)
    close(o, eo, bound(torch.float16, T, mo) + HALF_FLOOR, "o")
    close(s, es, state_bound(T, ms), "state")
    F.check_operators()


@pytest.mark.parametrize("T,dk,dv,hv", FAR)
def test_fp16_gradients_of_weight_that_lies_far_ahead(F, T, dk, dv, hv):  # noqa: F811
    """The same for the gradients: few tokens have one, and those far before them still feel it."""
    g = gen(72)
    q, k = (randn(g, 2, T, 2, dk) * 0.03).half(), (randn(g, 2, T, 2, dk) * 0.03).half()
    v = (randn(g, 2, T, hv, dv) * 200).half()
    go = sparse((randn(g, 2, T, 2, dv) * 200).half(), (50, 126))
    s0 = randn(g, 2, 2, dk, dv)
    ld, scale = torch.tensor([-0.7, -0.05], device="cuda"), 0.125
    got = F.linear_attention_backward(go, q, k, v, ld, scale=scale, initial_state=s0)
    exp = attention64(q, k, v, ld, scale, s0, None, go)
    maj = attention64(q, k, v, ld, scale, s0, None, go, absolute=True)
    for n, a, e, m in zip(("dq", "dk", "dv"), got, exp, maj):
        close(a, e, bound(torch.float16, T, m, 2) + HALF_FLOOR, n)
    lost = 2.0 ** -38 * scale * q.double().abs().amax() * go.double().abs().sum(1)[:, :, None]  # of q lam^t, times every gradient
    close(got[3], exp[3], state_bound(T, maj[3]) + lost, "ds0")
    F.check_operators()


@pytest.mark.parametrize("T", [256, 600])
def test_fp16_later_tokens_cost_earlier_ones_no_precision(F, T):  # noqa: F811
    """A token whose keys are at the type's upper end, after tokens whose keys are at its lower end."""
    g = gen(73)
    q = (randn(g, 1, T, 1, 64) * 2e4).clamp(-6e4, 6e4).half()
    k = (randn(g, 1, T, 1, 64) * 2.0 ** -14).half()
    v = randn(g, 1, T, 1, 64, dtype=torch.float16)
    ld, scale = torch.tensor([-0.01], device="cuda"), 0.125
    at = T - 100
    k[:, at:at + 3] = 6e4
    v[:, at:at + 3] *= 2.0 ** -14
    o = F.linear_attention(q, k, v, ld, scale=scale)[:, :at]
    eo, _ = attention64(q[:, :at], k[:, :at], v[:, :at], ld, scale)
    mo, _ = attention64(q[:, :at], k[:, :at], v[:, :at], ld, scale, absolute=True)
    close(o, eo, bound(torch.float16, T, mo) + HALF_FLOOR, "o")
    k[:, at] = float("inf")
    assert torch.equal(F.linear_attention(q, k, v, ld, scale=scale)[:, :at], o)


RINGS = [
    # rows enough for every team to fill each of its stages again; one to sixteen warps a row, with and without sums
    (torch.float32, (5453, 2048), None, True, True, True),
    (torch.float32, (2, 9000, 384), (2, 9000, 384), True, True, True),
    (torch.float32, (20000, 1024), None, False, False, False),
    (torch.float32, (3000, 8192), None, True, False, True),
    (torch.bfloat16, (4, 10000, 512), (4, 1, 512), True, True, True),
    (torch.float16, (6000, 4096), None, False, True, False),
]


@pytest.mark.parametrize("case", RINGS, ids=str)
def test_rows_keep_their_values_while_the_next_ones_land(F, case):  # noqa: F811
    """Stages of the rings are filled again only when they have been read: the same bits time after time, and the formula's values."""
    x, y, wp, wn, gate, s, gu, gn = norm_inputs(case)
    first = None
    for _ in range(25):
        got = []
        for save in ("full", "int8"):
            u, n, saved = F.gated_residual_norm(x, y, post_weight=wp, pre_weight=wn, gate=gate, residual_scale=s, save=save)
            got += [u, n, *F.gated_residual_norm_backward(gu, None if wn is None else gn, saved)]
        if first is None:
            first = got
        assert all(a is b is None or torch.equal(a, b) for a, b in zip(first, got))
    u, n = first[:2]
    e, e32 = UNIT[x.dtype], (x.shape[-1] + 16) * UNIT[torch.float32]
    exp, maj = norm64(x, y, wp, wn, gate, s, 1e-6)["u"]
    floor = HALF_FLOOR if x.dtype == torch.float16 else 0.0
    close(u, exp, e * exp.abs() + 2 * e32 * maj + floor, "u")
    if wn is not None:
        U = u.double()
        N = wn.double() * U / torch.sqrt((U * U).mean(-1, keepdim=True) + 1e-6)
        close(n, N, (e + e32) * N.abs() + floor + 1e-30, "n")
    F.check_operators()


def test_forward_mode_tangents_of_any_tensor_are_refused(F):  # noqa: F811
    """The kernels have no forward-mode form; results without the tangent would be derivatives of zero."""
    from lama_b200 import LamaError
    ad = torch.autograd.forward_ad
    z, ld, s = torch.randn(1, 4, 2, 8, device="cuda"), torch.zeros(2, device="cuda"), torch.zeros(1, 2, 8, 8, device="cuda")
    x, w = torch.randn(3, 8, device="cuda"), torch.ones(8, device="cuda")
    _, _, saved = F.gated_residual_norm(x, x, post_weight=w, pre_weight=w, save="full")
    with ad.dual_level():
        d, dx, dw, ds, dl = (ad.make_dual(t, torch.ones_like(t)) for t in (z, x, w, s, ld))
        for f in (lambda: F.linear_attention(z, d, z, ld), lambda: F.linear_attention(z, z, d[:, :, :1], ld),
                  lambda: F.linear_attention(z, z, z, dl), lambda: F.linear_attention(z, z, z, ld, initial_state=ds),
                  lambda: F.linear_attention_backward(d, z, z, z, ld), lambda: F.linear_attention_step(
                      z[:, 0], z[:, 0], z[:, 0], ld, ds),
                  lambda: F.gated_residual_norm(x, dx), lambda: F.gated_residual_norm(x, x, gate=dx),
                  lambda: F.gated_residual_norm(x, x, pre_weight=dw), lambda: F.gated_residual_norm(x, x, residual_scale=dw),
                  lambda: F.gated_residual_norm_backward(dx, x, saved)):
            with pytest.raises(LamaError) as ex:
                f()
            assert "forward-mode" in ex.value.msg
        with pytest.raises(Exception):  # in the autograd function torch itself refuses
            F.linear_attention(d, z.clone().requires_grad_(), z, ld)
    F.linear_attention(z, z, z, ld)


def test_a_step_is_seen_by_autograd(F):  # noqa: F811
    """A state that a graph saved and that a step then overwrote is an error in the backward pass, not a wrong gradient."""
    g = gen(74)
    q, k, v = (randn(g, 1, 5, 2, 16) for _ in range(3))
    ld, s = decays(2), randn(g, 1, 2, 16, 16)
    for out in (False, True):
        state = s.clone()
        o = F.linear_attention(q.clone().requires_grad_(), k, v, ld, initial_state=state)
        before = state._version
        with torch.no_grad():
            if out:
                F.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], ld, s, out_state=state)
            else:
                F.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], ld, state)
        assert state._version > before
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            o.sum().backward()
    with torch.inference_mode():  # such tensors have no versions
        state = s.clone()
        F.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], ld, state)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32], ids=str)
def test_training_is_the_same_with_and_without_the_final_state(F, dtype):  # noqa: F811
    g = gen(75)
    q, k, v, go = (randn(g, 2, 1100, 2, 64, dtype=dtype) for _ in range(4))
    got = []
    for state in (False, True):
        ts = [t.clone().requires_grad_() for t in (q, k, v)]
        out = F.linear_attention(*ts, decays(2), return_state=state)
        o = out[0] if state else out
        o.backward(go)
        got.append([o, *(t.grad for t in ts)])
    assert all(torch.equal(a, b) for a, b in zip(*got))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
def test_a_thread_s_first_call(F, dtype):  # noqa: F811
    """A thread that has made no CUDA call yet (autograd's own, at a process's first backward pass) runs the same kernels."""
    import threading
    g = gen(77)
    q, k, v, go = (randn(g, 2, 1100, 2, 64, dtype=dtype) for _ in range(4))
    ld = decays(2)

    def work():
        return [F.linear_attention(q, k, v, ld), *F.linear_attention_backward(go, q, k, v, ld)[:3]]
    exp = [t.clone() for t in work()]
    work()  # its memory stays with the allocator: the thread's call needs no other CUDA call
    for part in (work, lambda: [exp[0], *F.linear_attention_backward(go, q, k, v, ld)[:3]]):
        got = []
        t = threading.Thread(target=lambda: got.extend(part()))
        t.start()
        t.join()
        assert len(got) == 4 and all(torch.equal(a, b) for a, b in zip(got, exp))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32], ids=str)
def test_training_is_the_same_with_and_without_the_final_state(F, dtype):  # noqa: F811
    g = gen(75)
    q, k, v, go = (randn(g, 2, 1100, 2, 64, dtype=dtype) for _ in range(4))
    got = []
    for state in (False, True):
        ts = [t.clone().requires_grad_() for t in (q, k, v)]
        out = F.linear_attention(*ts, decays(2), return_state=state)
        o = out[0] if state else out
        o.backward(go)
        got.append([o, *(t.grad for t in ts)])
    assert all(torch.equal(a, b) for a, b in zip(*got))


# ------------------------------------------------------------------ the range's upper end

def chunked64(q, k, v, g, scale):
    """The recurrence in 64 bits, 256 tokens at a time: (o, final state), differentiable."""
    H = g.numel()
    q, k, v = (x.repeat_interleave(H // x.shape[2], 2).transpose(1, 2) for x in (q, k, v))
    gd = g.double()[None, :, None, None]
    s = q.new_zeros(q.shape[0], H, q.shape[-1], v.shape[-1])
    out = []
    for t in range(0, q.shape[2], 256):
        a, b, c = (x[:, :, t:t + 256] for x in (q, k, v))
        i = torch.arange(a.shape[2], device="cuda", dtype=torch.float64)
        d = (i[:, None] - i[None])[None, None]
        m = torch.where(d >= 0, torch.exp(gd * d.clamp_min(0)), 0.0)
        w = torch.exp(gd * (i[None, None, :, None] + 1))
        out.append(scale * (((a @ b.transpose(-1, -2)) * m) @ c + w * (a @ s)))
        s = torch.exp(gd * a.shape[2]) * s + (b * torch.exp(gd * (a.shape[2] - 1 - i[None, None, :, None]))).transpose(-1, -2) @ c
    return torch.cat(out, 2).transpose(1, 2), s


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32], ids=str)
@pytest.mark.parametrize("T,dk,dv", [(65536, 64, 64), (40001, 128, 80)])
def test_long_sequences(F, dtype, T, dk, dv):  # noqa: F811
    """A 2048x2048 image's latent, and an odd length; two heads of keys for four."""
    g = gen(76)
    q, k, v = randn(g, 1, T, 4, dk, dtype=dtype), randn(g, 1, T, 2, dk, dtype=dtype), randn(g, 1, T, 4, dv, dtype=dtype)
    go, gs = randn(g, 1, T, 4, dv, dtype=dtype), randn(g, 1, 4, dk, dv)
    ld, scale = decays(4), dk ** -0.5
    o, s = F.linear_attention(q, k, v, ld, return_state=True)
    got = F.linear_attention_backward(go, q, k, v, ld, grad_state=gs)
    sums = []
    for f in (lambda x: x.double(), lambda x: x.double().abs()):
        ts = [f(x).requires_grad_() for x in (q, k, v)]
        eo, es = chunked64(*ts, ld, scale)
        sums.append([eo.detach(), es.detach(), *torch.autograd.grad([eo, es], ts, [f(go), f(gs)])])
    exp, maj = sums
    floor = HALF_FLOOR if dtype == torch.float16 else 0.0
    close(o, exp[0], bound(dtype, T, maj[0]) + floor, "o")
    close(s, exp[1], state_bound(T, maj[1]), "state")
    for n, a, e, m in zip(("dq", "dk", "dv"), got, exp[2:], maj[2:]):
        close(a, e, bound(dtype, T, m, 4) + floor, n)
    F.check_operators()


@pytest.mark.parametrize("dtype,shape", [(torch.bfloat16, (5000, 3, 128)), (torch.float32, (1500, 2, 520)),
                                         (torch.float16, (700, 40, 257))], ids=str)
def test_a_gate_for_each_of_many_images(F, dtype, shape):  # noqa: F811
    """More gate rows than the kernels have CTAs: every one with its own sums."""
    case = (dtype, shape, (shape[0], 1, shape[2]), True, True, True)
    x, y, wp, wn, gate, s, gu, gn = norm_inputs(case)
    kw = dict(post_weight=wp, pre_weight=wn, residual_scale=s, save="full")
    u, n, saved = F.gated_residual_norm(x, y, gate=gate, **kw)
    g1 = F.gated_residual_norm_backward(gu, gn, saved)
    # a gate for each token holds the same numbers: the same rows, and its gradient summed over an image's tokens
    wide = gate.expand(shape).contiguous()
    u2, n2, saved = F.gated_residual_norm(x, y, gate=wide, **kw)
    g2 = F.gated_residual_norm_backward(gu, gn, saved)
    e, e32, rows = UNIT[dtype], 4 * (shape[2] + 32) * UNIT[torch.float32], shape[0] * shape[1]
    floor = HALF_FLOOR if dtype == torch.float16 else 0.0
    for a, b in ((u, u2), (n, n2), (g1.x, g2.x), (g1.y, g2.y)):
        # one order of the same products apart: a last place of the results where they round the other way
        close(a, b.double(), 2 * e * b.double().abs() + e32 * (b.double().abs() + 1) + floor)
    dg = g2.gate.double()
    close(g1.gate[:, 0], dg.sum(1), 2 * e * dg.abs().sum(1) + e32 * (dg.abs().sum(1) + 1) + floor * shape[1], "dgate")
    U = u.double()
    uh = U / torch.sqrt((U * U).mean(-1, keepdim=True) + 1e-6)
    t = gn.double() * uh
    close(g1.pre_weight, t.sum((0, 1)), (e32 + rows * 2.0 ** -23) * t.abs().sum((0, 1)), "dw_pre")


@pytest.mark.parametrize("T,dk,dv", [(100, 33, 33), (26, 33, 16), (1000, 33, 20), (128, 64, 64), (60, 128, 72)])
def test_bf16_results_are_rounded_once(F, T, dk, dv):  # noqa: F811
    """Where the scores and what is carried keep 16 bits or more (heads of any odd size, and a chunk of the others) a result is
    its sum rounded once: e |result|, and 2^-16 M for the two parts beside the fp32 sums."""
    g = gen(78)
    q, k, v, go = (randn(g, 2, T, 2, d, dtype=torch.bfloat16) for d in (dk, dk, dv, dv))
    ld, scale = decays(2), dk ** -0.5
    got = F.linear_attention(q, k, v, ld), *F.linear_attention_backward(go, q, k, v, ld)[:3]
    exp = attention64(q, k, v, ld, scale)[:1] + attention64(q, k, v, ld, scale, None, None, go)[:3]
    maj = attention64(q, k, v, ld, scale, absolute=True)[:1] + attention64(q, k, v, ld, scale, None, None, go, absolute=True)[:3]
    e = UNIT[torch.bfloat16]
    for n, a, x, m in zip(("o", "dq", "dk", "dv"), got, exp, maj):
        close(a, x, e * x.abs() + 2.0 ** -16 * m + bound(torch.float32, T, m, 2), n)
