"""The token-mixer operators (lama_b200.operators, no counterpart in the reference) against plain
64-bit implementations.

Bounds are per element and come from rounding alone.  With a result written as a sum of products, M
is the same sum over absolute values; every rounding to a type with unit e (half a unit in the last
place, relative) moves an element by at most e * M.  For 16-bit inputs two roundings reach each term
of the attention's results (that of the scores or of the carried state, and the result's), so the
bound is 2 e M.  For 32-bit inputs the sums are what counts: up to N = 128 + 2 * 128 + chunks
terms added one after another in fp32, twice that for the parts a product is split into, so the bound
is 2 N 2^-24 M.
"""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
TYPES = [torch.bfloat16, torch.float16, torch.float32]


@pytest.fixture(scope="module")
def F():
    from lama_b200 import operators
    return operators


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def randn(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


def close(got, exp, bound, what=""):
    d = (got.double() - exp).abs()
    bad = ~(d <= bound)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((d / bound.clamp_min(1e-300)).max()):.3g} bounds"


# ------------------------------------------------------------------ linear attention

def attention64(q, k, v, g, scale, s0=None, lengths=None, go=None, gs=None, absolute=False):
    """The sums written out in 64 bits: (o, state) or, with go, (dq, dk, dv, ds0)."""
    B, T = q.shape[:2]
    H = g.numel()
    f = (lambda x: x.double().abs()) if absolute else (lambda x: x.double())
    heads = lambda x: f(x).repeat_interleave(H // x.shape[2], 2).transpose(1, 2)  # noqa: E731
    Q, K, V = heads(q), heads(k), heads(v)
    pos = torch.arange(T, device="cuda", dtype=torch.float64)
    lens = torch.full((B,), T, device="cuda") if lengths is None else lengths.clamp(0, T)
    on = (pos[None] < lens[:, None]).double()[:, None, :, None]
    Q, K, V = Q * on, K * on, V * on
    gd = g.double()[None, :, None, None]

    def lam(n):
        return torch.where(n == 0, 1.0, torch.exp(gd * n.clamp_min(1)))
    dist = (pos[:, None] - pos[None, :])[None, None]
    m = torch.where(dist >= 0, lam(dist.clamp_min(0)), 0.0)
    w_in = lam(pos[None, None, :, None] + 1)
    left = (lens[:, None, None, None] - 1 - pos[None, None, :, None])
    w_out = torch.where(left >= 0, lam(left.clamp_min(0)), 0.0)
    w_all = lam(lens.double()[:, None, None, None])
    S = torch.zeros(B, H, q.shape[-1], v.shape[-1], dtype=torch.float64, device="cuda") if s0 is None else f(s0)
    scale = abs(scale) if absolute else scale
    A = (Q @ K.transpose(-1, -2)) * m
    if go is None:
        o = scale * (A @ V + w_in * (Q @ S)) * on
        return o.transpose(1, 2), (K * w_out).transpose(-1, -2) @ V + w_all * S
    G = f(go).transpose(1, 2) * on
    D = torch.zeros_like(S) if gs is None else f(gs)
    P = (G @ V.transpose(-1, -2)) * m
    dq = scale * (P @ K + w_in * (G @ S.transpose(-1, -2)))
    dk = scale * P.transpose(-1, -2) @ Q + w_out * (V @ D.transpose(-1, -2))
    dv = scale * A.transpose(-1, -2) @ G + w_out * (K @ D)
    ds = scale * (Q * w_in).transpose(-1, -2) @ G + w_all * D

    def back(x, like):
        x = (x * on).transpose(1, 2)
        return x.reshape(B, T, like.shape[2], H // like.shape[2], x.shape[-1]).sum(3)
    return back(dq, q), back(dk, k), back(dv, v), ds


def bound(dtype, T, M, heads=1):
    n = 2 * (128 + 256 + (T + 127) // 128 + heads) * UNIT[torch.float32]
    return (n if dtype == torch.float32 else n + 2 * UNIT[dtype]) * M + 1e-30


def state_bound(T, M):
    return 2 * (128 + (T + 127) // 128 + 8) * UNIT[torch.float32] * M + 1e-30


def decays(h):
    return torch.tensor([-0.7 * (3e-4 / 0.7) ** (i / max(h - 1, 1)) for i in range(h)], device="cuda")


CASES = [
    # dtype, B, T, H, dk, dv, heads of q, k, v, ragged, state
    (torch.bfloat16, 2, 200, 3, 64, 64, 3, 3, 3, False, True),
    (torch.bfloat16, 1, 1, 2, 64, 64, 2, 2, 2, False, True),
    (torch.bfloat16, 1, 127, 1, 128, 128, 1, 1, 1, False, False),
    (torch.bfloat16, 1, 129, 2, 128, 64, 2, 1, 2, False, True),
    (torch.bfloat16, 3, 385, 4, 64, 128, 2, 2, 4, True, True),
    (torch.bfloat16, 2, 1100, 2, 33, 16, 2, 2, 1, True, False),
    (torch.bfloat16, 1, 2500, 2, 80, 80, 2, 2, 2, False, True),
    (torch.float16, 2, 300, 2, 64, 64, 2, 2, 2, False, True),
    (torch.float16, 1, 140, 4, 128, 80, 1, 2, 4, True, True),
    (torch.float16, 2, 1000, 2, 16, 33, 2, 2, 2, False, False),
    (torch.float32, 2, 257, 2, 64, 64, 2, 2, 2, False, True),
    (torch.float32, 1, 1500, 4, 128, 128, 4, 2, 1, True, True),
    (torch.float32, 2, 130, 2, 33, 80, 2, 1, 2, False, False),
    (torch.float32, 3, 5, 1, 1, 1, 1, 1, 1, True, True),
]


def attention_inputs(case, seed=7):
    dtype, B, T, H, dk, dv, hq, hk, hv, ragged, state = case
    g = gen(seed)
    q, k, v = randn(g, B, T, hq, dk, dtype=dtype), randn(g, B, T, hk, dk, dtype=dtype), randn(g, B, T, hv, dv, dtype=dtype)
    s0 = randn(g, B, H, dk, dv) * 2 if state else None
    lengths = None
    if ragged:
        lengths = torch.randint(0, T + 1, (B,), generator=g, device="cuda", dtype=torch.int32)
        lengths[0] = 0  # a sequence of nothing
    return g, q, k, v, decays(H), dk ** -0.5, s0, lengths


@pytest.mark.parametrize("case", CASES, ids=str)
def test_attention_matches_the_sums(F, case):
    _, q, k, v, ld, scale, s0, lengths = attention_inputs(case)
    o, s = F.linear_attention(q, k, v, ld, initial_state=s0, lengths=lengths, return_state=True)
    eo, es = attention64(q, k, v, ld, scale, s0, lengths)
    mo, ms = attention64(q, k, v, ld, scale, s0, lengths, absolute=True)
    close(o, eo, bound(q.dtype, q.shape[1], mo), "o")
    close(s, es, state_bound(q.shape[1], ms), "state")
    F.check_operators()


@pytest.mark.parametrize("case", CASES, ids=str)
def test_attention_gradients_match_the_formula(F, case):
    g, q, k, v, ld, scale, s0, lengths = attention_inputs(case)
    go = randn(g, *q.shape[:2], ld.numel(), v.shape[-1], dtype=q.dtype)
    gs = randn(g, q.shape[0], ld.numel(), q.shape[-1], v.shape[-1])
    got = F.linear_attention_backward(go, q, k, v, ld, initial_state=s0, lengths=lengths, grad_state=gs)
    exp = attention64(q, k, v, ld, scale, s0, lengths, go, gs)
    maj = attention64(q, k, v, ld, scale, s0, lengths, go, gs, absolute=True)
    for n, a, e, m in zip(("dq", "dk", "dv"), got, exp, maj):
        close(a, e, bound(q.dtype, q.shape[1], m, ld.numel()), n)
    if s0 is None:
        assert got[3] is None
    else:
        close(got[3], exp[3], state_bound(q.shape[1], maj[3]), "ds0")
    F.check_operators()


def test_attention_gradients_match_differences(F):
    """L = <w, o> + <z, state> is linear in each of q, k, v and the initial state alone, so a central
    difference of any width is its directional derivative; both sides err by their fp32 sums."""
    g, q, k, v, ld, scale, s0, _ = attention_inputs((torch.float32, 2, 300, 2, 64, 64, 1, 2, 1, False, True))
    w, z = randn(g, 2, 300, 2, 64), randn(g, 2, 2, 64, 64)
    grads = F.linear_attention_backward(w, q, k, v, ld, initial_state=s0, grad_state=z)
    args = [q, k, v, s0]

    def loss(a):
        o, s = F.linear_attention(a[0], a[1], a[2], ld, initial_state=a[3], return_state=True)
        return float((o.double() * w).sum() + (s.double() * z).sum())
    for i in range(4):
        d = randn(g, *args[i].shape)
        up, dn = list(args), list(args)
        up[i], dn[i] = args[i] + d, args[i] - d
        diff = (loss(up) - loss(dn)) / 2
        big = list(args)
        big[i] = args[i].abs() + d.abs()
        mo, ms = attention64(*big[:3], ld, scale, big[3], absolute=True)
        tol = float((bound(torch.float32, 300, mo, 2) * w.abs()).sum() + (state_bound(300, ms) * z.abs()).sum())
        assert abs(diff - float((grads[i].double() * d).sum())) <= 2 * tol


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_attention_takes_any_strides(F, dtype):
    """Packed projections, transposed heads, odd offsets and a reversed batch read like contiguous copies."""
    g = gen(3)
    B, T, H, D = 2, 150, 2, 64
    packed = randn(g, B, T, 3, H, D, dtype=dtype)
    odd = randn(g, B * T * H * D + 1, dtype=dtype)[1:].view(B, T, H, D)  # not 16-byte aligned
    swapped = randn(g, B, H, T, D, dtype=dtype).transpose(1, 2)
    shared = randn(g, B, 1, 1, D, dtype=dtype).expand(B, T, 1, D)
    last = randn(g, B, T, D, H, dtype=dtype).transpose(2, 3)
    ld = decays(H)
    for q, k, v in ((packed[:, :, 0], packed[:, :, 1], packed[:, :, 2]), (odd, swapped, packed[:, :, 1]),
                    (swapped, odd, odd), (packed[:, ::2].repeat(1, 2, 1, 1, 1)[:, :T, 0], shared, last)):
        a = F.linear_attention(q, k, v, ld)
        b = F.linear_attention(q.contiguous(), k.contiguous(), v.contiguous(), ld)
        assert torch.equal(a, b)
        ga = F.linear_attention_backward(a.transpose(1, 2).contiguous().transpose(1, 2), q, k, v, ld)
        gb = F.linear_attention_backward(b, q.contiguous(), k.contiguous(), v.contiguous(), ld)
        for x, y in zip(ga[:3], gb[:3]):
            assert torch.equal(x, y)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_a_sequence_in_pieces_equals_the_whole(F, dtype):
    """The carried state is exact up to fp32 sums, so strips fed one after another give the whole's outputs."""
    _, q, k, v, ld, scale, s0, _ = attention_inputs((dtype, 2, 700, 2, 64, 64, 2, 2, 2, False, True))
    o, s = F.linear_attention(q, k, v, ld, initial_state=s0, return_state=True)
    mo, ms = attention64(q, k, v, ld, scale, s0, absolute=True)
    state, parts = s0, []
    for a, b in ((0, 1), (1, 130), (130, 500), (500, 700)):
        p, state = F.linear_attention(q[:, a:b], k[:, a:b], v[:, a:b], ld, initial_state=state, return_state=True)
        parts.append(p)
    close(torch.cat(parts, 1), o.double(), 2 * bound(dtype, 700, mo), "o")
    close(state, s.double(), 2 * state_bound(700, ms), "state")


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_extreme_decays(F, dtype):
    """No memory (-inf, and a decay that underflows), none forgotten (0)."""
    g = gen(5)
    q, k, v = (randn(g, 1, 300, 3, 64, dtype=dtype) for _ in range(3))
    ld = torch.tensor([-math.inf, -200.0, 0.0], device="cuda")
    s0 = randn(g, 1, 3, 64, 64)
    o, s = F.linear_attention(q, k, v, ld, initial_state=s0, return_state=True)
    eo, es = attention64(q, k, v, ld, 0.125, s0)
    mo, ms = attention64(q, k, v, ld, 0.125, s0, absolute=True)
    close(o, eo, bound(dtype, 300, mo))
    close(s, es, state_bound(300, ms))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_tokens_past_a_length_are_not_read(F, dtype):
    g = gen(6)
    q, k, v, go = (randn(g, 3, 300, 2, 64, dtype=dtype) for _ in range(4))
    lengths = torch.tensor([0, 131, 300], device="cuda", dtype=torch.int32)
    ld = decays(2)
    o, s = F.linear_attention(q, k, v, ld, lengths=lengths, return_state=True)
    grads = F.linear_attention_backward(go, q, k, v, ld, lengths=lengths)
    for fill in (math.nan, math.inf, torch.finfo(dtype).min):
        bad = [x.clone() for x in (q, k, v, go)]
        for x in bad:
            x[0], x[1, 131:] = fill, fill
        o2, s2 = F.linear_attention(*bad[:3], ld, lengths=lengths, return_state=True)
        assert torch.equal(o, o2) and torch.equal(s, s2)
        for a, b in zip(grads[:3], F.linear_attention_backward(bad[3], *bad[:3], ld, lengths=lengths)[:3]):
            assert torch.equal(a, b)
    assert not o[0].any() and not o[1, 131:].any() and not s[0].any()
    # lengths outside the sequence are clamped
    wide = torch.tensor([-5, 131, 9999], device="cuda", dtype=torch.int32)
    assert torch.equal(F.linear_attention(q, k, v, ld, lengths=wide), o)


def test_large_fp16_values_do_not_overflow_inside(F):
    """Scores and states above fp16's 65504 whose outputs fit."""
    g = gen(9)
    q = (randn(g, 1, 300, 1, 64).abs() * 300).half()
    k = (randn(g, 1, 300, 1, 64).abs() * 300).half()
    v = (randn(g, 1, 300, 1, 64) * 1e-4).half()
    ld = torch.tensor([-1e-3], device="cuda")
    o = F.linear_attention(q, k, v, ld)
    eo, _ = attention64(q, k, v, ld, 0.125)
    mo, _ = attention64(q, k, v, ld, 0.125, absolute=True)
    close(o, eo, bound(torch.float16, 300, mo))


def test_results_do_not_change_from_run_to_run(F):
    _, q, k, v, ld, _, s0, _ = attention_inputs((torch.bfloat16, 2, 2000, 4, 64, 64, 2, 4, 1, False, True))
    a = F.linear_attention(q, k, v, ld, initial_state=s0, return_state=True)
    ga = F.linear_attention_backward(a[0], q, k, v, ld, initial_state=s0)
    for _ in range(3):
        b = F.linear_attention(q, k, v, ld, initial_state=s0, return_state=True)
        assert all(torch.equal(x, y) for x, y in zip(a, b))
        gb = F.linear_attention_backward(a[0], q, k, v, ld, initial_state=s0)
        assert all(torch.equal(x, y) for x, y in zip(ga, gb))


def test_attention_autograd(F):
    _, q, k, v, ld, scale, s0, _ = attention_inputs((torch.float32, 1, 200, 2, 64, 64, 2, 1, 2, False, True))
    for t in (q, k, v, s0):
        t.requires_grad_()
    o, s = F.linear_attention(q, k, v, ld, initial_state=s0, return_state=True)
    w, z = torch.ones_like(o), torch.full_like(s, 0.5)
    ((o * w).sum() + (s * z).sum()).backward()
    exp = F.linear_attention_backward(w, q.detach(), k.detach(), v.detach(), ld, initial_state=s0.detach(), grad_state=z)
    for t, e in zip((q, k, v, s0), exp):
        assert torch.equal(t.grad, e)
    q.grad = None
    F.linear_attention(q, k, v, ld).sum().backward()
    assert torch.isfinite(q.grad).all()


def test_empty_sequences(F):
    z = torch.zeros(2, 0, 3, 64, device="cuda", dtype=torch.bfloat16)
    s0 = torch.ones(2, 3, 64, 64, device="cuda")
    o, s = F.linear_attention(z, z, z, decays(3), initial_state=s0, return_state=True)
    assert o.shape == (2, 0, 3, 64) and torch.equal(s, s0)
    dq, dk, dv, ds = F.linear_attention_backward(o, z, z, z, decays(3), initial_state=s0, grad_state=s0)
    assert dq.shape == z.shape and torch.equal(ds, s0)


def test_attention_on_a_side_stream(F):
    _, q, k, v, ld, _, _, _ = attention_inputs((torch.bfloat16, 1, 1500, 2, 64, 64, 2, 2, 2, False, False))
    exp = F.linear_attention(q, k, v, ld)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = F.linear_attention(q, k, v, ld)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, exp)


# ------------------------------------------------------------------ single tokens

@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("shape", [(1, 2, 64, 64, 2, 2, 2), (5, 4, 128, 128, 2, 4, 1), (3, 2, 33, 17, 2, 1, 2),
                                   (2, 1, 1, 1, 1, 1, 1), (4, 3, 80, 36, 3, 3, 3)], ids=str)
def test_step_matches_the_recurrence(F, dtype, shape):
    B, H, dk, dv, hq, hk, hv = shape
    g = gen(11)
    q, k, v = randn(g, B, hq, dk, dtype=dtype), randn(g, B, hk, dk, dtype=dtype), randn(g, B, hv, dv, dtype=dtype)
    state, ld, scale = randn(g, B + 3, H, dk, dv) * 3, decays(H), 0.3
    slots = torch.randperm(B + 3, generator=g, device="cuda")[:B].to(torch.int32)
    if B > 1:
        slots[1] = -1
    if B > 2:
        slots[2] = B + 3
    before = state.clone()
    out = state.clone()
    o1 = F.linear_attention_step(q, k, v, ld, state, scale=scale, slots=slots, out_state=out)
    assert torch.equal(state, before)
    o2 = F.linear_attention_step(q, k, v, ld, state, scale=scale, slots=slots)
    assert torch.equal(o1, o2) and torch.equal(out, state)
    lam = torch.exp(ld.double())[:, None, None]
    e = UNIT[torch.float32] * 4
    for b in range(B):
        s = int(slots[b])
        if not 0 <= s < B + 3:
            assert not o1[b].any()
            continue
        Q, K, V = (x[b].double().repeat_interleave(H // x.shape[1], 0) for x in (q, k, v))
        S = lam * before[s].double() + K[:, :, None] * V[:, None]
        M = lam * before[s].double().abs() + (K[:, :, None] * V[:, None]).abs()
        close(state[s], S, e * M)
        mo = scale * (Q.abs()[:, :, None] * M).sum(1)
        close(o1[b], scale * (Q[:, :, None] * S).sum(1), (UNIT[dtype] + (dk + 8) * UNIT[torch.float32]) * mo)
        before[s] = state[s].clone()
    untouched = torch.ones(B + 3, dtype=torch.bool, device="cuda")
    untouched[slots[(slots >= 0) & (slots < B + 3)].long()] = False
    assert torch.equal(state[untouched], before[untouched])


def test_steps_continue_a_prompt(F):
    _, q, k, v, ld, scale, _, _ = attention_inputs((torch.float32, 2, 140, 2, 64, 64, 2, 2, 2, False, False))
    o = F.linear_attention(q, k, v, ld)
    mo, _ = attention64(q, k, v, ld, scale, absolute=True)
    _, s = F.linear_attention(q[:, :130], k[:, :130], v[:, :130], ld, return_state=True)
    for t in range(130, 140):
        got = F.linear_attention_step(q[:, t], k[:, t], v[:, t], ld, s)
        close(got, o[:, t].double(), 2 * bound(torch.float32, 140, mo)[:, t])


# ------------------------------------------------------------------ 8-bit checkpoints

def values8(x):
    """The checkpoint's definition, each operation one fp32 rounding."""
    c = x.shape[-1]
    g = -(-c // 128)
    p = torch.nn.functional.pad(x.float(), (0, g * 128 - c)).view(*x.shape[:-1], g, 128)
    a = p.abs().amax(-1, keepdim=True)
    zero, top = a < 2.0 ** -96, torch.full_like(a, 127.0)  # a tensor: torch divides by a number in two roundings
    codes = torch.round(p * torch.where(zero, 0.0, top / a))
    v = codes * torch.where(zero, 0.0, a / top)
    v = torch.where(torch.isfinite(a), v, math.nan)
    return v.flatten(-2)[..., :c].to(x.dtype)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("shape", [(1, 1), (3, 128), (7, 397), (130, 512), (2, 3, 1000), (5, 8), (2, 4100)], ids=str)
def test_checkpoint_holds_the_defined_values(F, dtype, shape):
    x = (randn(gen(1), *shape) * torch.exp(randn(gen(2), shape[-1]) * 2)).to(dtype)
    c = F.checkpoint_store(x)
    assert c.codes.shape == x.shape and c.codes.dtype == torch.int8
    assert torch.equal(F.checkpoint_restore(c), values8(x))
    a = F.checkpoint_restore(c, torch.float32)
    assert torch.equal(a.to(dtype), values8(x))


def test_checkpoint_of_odd_values(F):
    x = torch.zeros(8, 256, device="cuda")
    x[1, 3], x[2, 5], x[3, 200] = math.nan, math.inf, -math.inf
    x[4] = 1e-35
    x[5] = torch.finfo(torch.float32).max  # 127 (a / 127) may round past the type's end there
    x[6, :128] = 1e-40
    x[7] = torch.linspace(-1, 1, 256)
    got = F.checkpoint_restore(F.checkpoint_store(x))
    assert torch.equal(torch.nan_to_num(got, 7), torch.nan_to_num(values8(x), 7))
    assert torch.isnan(got[1, :128]).all() and not got[1, 128:].any() and torch.isnan(got[3, 128:]).all()
    top = torch.full((1, 128), torch.finfo(torch.bfloat16).max, device="cuda", dtype=torch.bfloat16)
    assert torch.equal(F.checkpoint_restore(F.checkpoint_store(top)), top)
    part = torch.randn(9, 300, device="cuda")
    for v in (part[:, 3:200], part[::2], part.t(), part[0], part[:, :0], part[:0]):
        assert torch.equal(F.checkpoint_restore(F.checkpoint_store(v)), values8(v) if v.numel() else v)


# ------------------------------------------------------------------ norms, gate and residual

def norm64(x, y, wp, wn, gate, s, eps, gu=None, gn=None, yk=None, uk=None):
    """The formulas in 64 bits, u rounded as defined; and majorants of every result."""
    X, Y = x.double(), y.double()
    C = x.shape[-1]
    G = torch.ones((), dtype=torch.float64, device="cuda") if gate is None else gate.double()
    S = s.double() if isinstance(s, torch.Tensor) else torch.tensor(float(s), dtype=torch.float64, device="cuda")
    WP = torch.ones(C, dtype=torch.float64, device="cuda") if wp is None else wp.double()
    ry = torch.ones_like(Y[..., :1]) if wp is None else 1 / torch.sqrt((Y * Y).mean(-1, keepdim=True) + eps)
    u = X + S * G * WP * Y * ry
    out = {"u": (u, X.abs() + (S * G * WP * Y * ry).abs())}
    if gu is None and gn is None:
        return out
    return out, ry, G, S, WP


NORMS = [
    # dtype, shape, gate shape, post, pre, scale vector
    (torch.bfloat16, (2, 37, 512), (2, 1, 512), True, True, True),
    (torch.bfloat16, (3, 5, 128), (3, 5, 128), True, True, False),
    (torch.bfloat16, (1, 300, 384), (384,), True, True, True),
    (torch.bfloat16, (2, 9, 2048), None, True, True, True),
    (torch.bfloat16, (40, 3, 257), (40, 1, 257), True, True, True),
    (torch.float16, (2, 33, 1000), (2, 1, 1000), True, True, True),
    (torch.float16, (1, 1, 16), (1, 1, 16), False, True, True),
    (torch.float32, (2, 50, 384), (2, 50, 384), True, True, True),
    (torch.float32, (700, 64), None, True, False, True),
    (torch.float32, (3, 7, 1), (3, 1, 1), True, True, True),
    (torch.float32, (2, 6, 5000), (2, 1, 5000), True, True, True),
    (torch.bfloat16, (3, 12000), None, False, True, False),
    (torch.float32, (4, 11, 96), (4, 1, 96), False, False, True),
]


def norm_inputs(case):
    dtype, shape, gshape, post, pre, vec = case
    g = gen(21)
    C = shape[-1]
    chan = torch.exp(randn(g, C) * 0.7)
    x, y = (randn(g, *shape) * chan).to(dtype), randn(g, *shape, dtype=dtype)
    wp = 1 + 0.2 * randn(g, C) if post else None
    wn = 1 + 0.2 * randn(g, C) if pre else None
    gate = None if gshape is None else randn(g, *gshape, dtype=dtype)
    s = 0.5 + 0.1 * randn(g, C) if vec else 0.7
    gu, gn = randn(g, *shape, dtype=dtype), randn(g, *shape, dtype=dtype)
    return x, y, wp, wn, gate, s, gu, gn


@pytest.mark.parametrize("save", [None, "full", "int8"])
@pytest.mark.parametrize("case", NORMS, ids=str)
def test_norm_matches_the_formula(F, case, save):
    x, y, wp, wn, gate, s, _, _ = norm_inputs(case)
    res = F.gated_residual_norm(x, y, post_weight=wp, pre_weight=wn, gate=gate, residual_scale=s, save=save)
    u, n = res[:2]
    C = x.shape[-1]
    e, e32 = UNIT[x.dtype], (C + 16) * UNIT[torch.float32]
    exp, maj = norm64(x, y, wp, wn, gate, s, 1e-6)["u"]
    close(u, exp, e * exp.abs() + 2 * e32 * maj, "u")  # one rounding of the sum, the statistics' fp32 sums
    if wn is None:
        assert n is None
    else:
        U = u.double()  # n is the norm of the rounded u
        N = wn.double() * U / torch.sqrt((U * U).mean(-1, keepdim=True) + 1e-6)
        close(n, N, (e + e32) * N.abs() + 1e-30, "n")
    if save == "int8":
        assert torch.equal(F.checkpoint_restore(res[2].y), values8(y))
        if wn is not None:
            assert torch.equal(F.checkpoint_restore(res[2].u), values8(u))
            assert res[2].nbytes < (y.nbytes + u.nbytes) or x.shape[-1] < 64


@pytest.mark.parametrize("save", ["full", "int8"])
@pytest.mark.parametrize("case", NORMS, ids=str)
def test_norm_gradients_match_the_formula(F, case, save):
    """Against the formulas in 64 bits at the values the checkpoint holds.  M sums absolute values of each
    formula's terms; statistics and column sums err by their number of fp32 terms, results by one rounding."""
    x, y, wp, wn, gate, s, gu, gn = norm_inputs(case)
    u, n, saved = F.gated_residual_norm(x, y, post_weight=wp, pre_weight=wn, gate=gate, residual_scale=s, save=save)
    got = F.gated_residual_norm_backward(gu, None if wn is None else gn, saved)
    C, rows = x.shape[-1], x.numel() // x.shape[-1]
    Y, U = y.double(), u.double()
    ry = torch.ones_like(Y[..., :1]) if wp is None else 1 / torch.sqrt((Y * Y).mean(-1, keepdim=True) + 1e-6)
    ru = 1 / torch.sqrt((U * U).mean(-1, keepdim=True) + 1e-6)
    if save == "int8":  # fp32 values, as the backward pass reads them
        Y = F.checkpoint_restore(saved.y, torch.float32).double()
        U = U if wn is None else F.checkpoint_restore(saved.u, torch.float32).double()
    G = torch.ones((), dtype=torch.float64, device="cuda") if gate is None else gate.double()
    S = s.double() if isinstance(s, torch.Tensor) else torch.tensor(float(s), dtype=torch.float64, device="cuda")
    WP = torch.ones(C, dtype=torch.float64, device="cuda") if wp is None else wp.double()
    e, e32 = UNIT[x.dtype], 4 * (C + 32) * UNIT[torch.float32]
    D, MD = gu.double(), gu.double().abs()
    if wn is not None:
        uh, wd = U * ru, wn.double() * gn.double()
        c, mc = (uh * wd).mean(-1, keepdim=True), (uh * wd).abs().mean(-1, keepdim=True)
        D, MD = D + ru * (wd - uh * c), MD + ru * (wd.abs() + uh.abs() * mc)
        dwn = (gn.double() * uh).flatten(0, -2).sum(0)
        close(got.pre_weight, dwn, (e32 + rows * 2.0 ** -23) * (gn.double() * uh).abs().flatten(0, -2).sum(0), "dw_pre")
    close(got.x, D, e * D.abs() + e32 * MD, "dx")
    yh = Y * ry
    dp, mdp = D * S * G, MD * (S * G).abs()
    if wp is None:
        close(got.y, dp, e * dp.abs() + e32 * mdp, "dy")
        assert got.post_weight is None
    else:
        c, mc = (yh * WP * dp).mean(-1, keepdim=True), (yh * WP).abs().mul(mdp).mean(-1, keepdim=True)
        dy, mdy = ry * (WP * dp - yh * c), ry * (WP.abs() * mdp + yh.abs() * mc)
        close(got.y, dy, e * dy.abs() + e32 * mdy, "dy")
        close(got.post_weight, (dp * yh).flatten(0, -2).sum(0),
              (e32 + rows * 2.0 ** -23) * (mdp * yh.abs()).flatten(0, -2).sum(0), "dw_post")
    if isinstance(s, torch.Tensor):
        close(got.residual_scale, (D * G * WP * yh).flatten(0, -2).sum(0),
              (e32 + rows * 2.0 ** -23) * (MD * (G * WP * yh).abs()).flatten(0, -2).sum(0) + 1e-30, "ds")
    if gate is not None:
        dg, mg = D * S * WP * yh, MD * (S * WP * yh).abs()
        red = [i for i in range(x.dim()) if i < x.dim() - gate.dim() or gate.shape[i - x.dim()] == 1 != x.shape[i]]
        if red:
            dg, mg = dg.sum(red).view(gate.shape), mg.sum(red).view(gate.shape)
        close(got.gate, dg, e * dg.abs() + (e32 + rows * 2.0 ** -23) * mg + 1e-30, "dgate")


def test_norm_gradients_match_differences(F):
    """Central differences of width h along random directions: off by h^2/6 of the third derivative, which for
    these unit-scale inputs (h = 0.01, directions of unit size per element) is below 1e-3 of the loss's scale."""
    x, y, wp, wn, gate, s, gu, gn = norm_inputs((torch.float32, (2, 6, 128), (2, 1, 128), True, True, True))
    names = ["x", "y", "post_weight", "pre_weight", "gate", "residual_scale"]
    vals = [x, y, wp, wn, gate, s]

    def loss(v):
        u, n = F.gated_residual_norm(v[0], v[1], post_weight=v[2], pre_weight=v[3], gate=v[4], residual_scale=v[5])
        return float((u.double() * gu).sum() + (n.double() * gn).sum())
    _, _, saved = F.gated_residual_norm(x, y, post_weight=wp, pre_weight=wn, gate=gate, residual_scale=s, save="full")
    g = F.gated_residual_norm_backward(gu, gn, saved)
    rng, h = gen(4), 0.01
    for i, name in enumerate(names):
        d = randn(rng, *vals[i].shape)
        up, dn = list(vals), list(vals)
        up[i], dn[i] = vals[i] + h * d, vals[i] - h * d
        diff = (loss(up) - loss(dn)) / (2 * h)
        exact = float((getattr(g, name).double() * d).sum())
        size = float((getattr(g, name).double() * d).abs().sum())
        assert abs(diff - exact) <= 1e-3 * size, name


@pytest.mark.parametrize("save", ["full", "int8"])
def test_norm_autograd(F, save):
    x, y, wp, wn, gate, s, gu, gn = norm_inputs((torch.bfloat16, (2, 50, 512), (2, 1, 512), True, True, True))
    kw = dict(post_weight=wp, pre_weight=wn, gate=gate, residual_scale=s)
    u, n, saved = F.gated_residual_norm(x, y, save=save, **kw)
    exp = F.gated_residual_norm_backward(gu, gn, saved)
    leaves = [t.requires_grad_() for t in (x, y, wp, wn, gate, s)]
    u2, n2, none = F.gated_residual_norm(x, y, save=save, **kw)
    assert none is None and torch.equal(u, u2) and torch.equal(n, n2)
    torch.autograd.backward([u2, n2], [gu, gn])
    for t, e in zip(leaves, exp):
        assert torch.equal(t.grad, e)
    for t in leaves:
        t.grad = None
    u3, n3, _ = F.gated_residual_norm(x, y, save=save, **kw)
    u3.sum().backward()  # no gradient of n
    assert torch.isfinite(x.grad).all() and not wn.grad.any()


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_norm_takes_strides_and_offsets(F, dtype):
    g = gen(8)
    big = randn(g, 2, 40, 600, dtype=dtype)
    x, y, gate = big[..., 3:403], big[:, :, 100:500], big[:, :1, 7:407]
    w = 1 + 0.1 * randn(g, 400)
    a = F.gated_residual_norm(x, y, post_weight=w, pre_weight=w, gate=gate, save="int8")
    b = F.gated_residual_norm(x.contiguous(), y.contiguous(), post_weight=w, pre_weight=w, gate=gate.contiguous(),
                              save="int8")
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    ga = F.gated_residual_norm_backward(big[..., 9:409], y, a[2])
    gb = F.gated_residual_norm_backward(big[..., 9:409].contiguous(), y.contiguous(), b[2])
    for p, q in zip(ga, gb):
        assert p is q is None or torch.equal(p, q)


def test_norm_of_zeros_and_of_nothing(F):
    z = torch.zeros(4, 64, device="cuda")
    w = torch.ones(64, device="cuda")
    u, n, saved = F.gated_residual_norm(z, z, post_weight=w, pre_weight=w, save="int8")
    assert not u.any() and not n.any()
    g = F.gated_residual_norm_backward(z + 1, z, saved)
    assert torch.equal(g.x, z + 1) and torch.isfinite(g.y).all()
    e = torch.zeros(0, 64, device="cuda")
    u, n, saved = F.gated_residual_norm(e, e, post_weight=w, pre_weight=w, save="full")
    g = F.gated_residual_norm_backward(e, e, saved)
    assert g.x.shape == (0, 64) and not g.pre_weight.any()


# ------------------------------------------------------------------ without the final state, and refusals

@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("dk,dv", [(64, 64), (128, 128), (128, 64), (64, 128)])
def test_long_sequences_cut_into_segments_without_a_final_state(F, dtype, dk, dv):
    """Few heads and many tokens: the states of segments are made and scanned, forward and backward."""
    g = gen(31)
    q, k, v, go = (randn(g, 1, 3000, 2, d, dtype=dtype) for d in (dk, dk, dv, dv))
    ld, scale = decays(2), dk ** -0.5
    o = F.linear_attention(q, k, v, ld)
    eo, _ = attention64(q, k, v, ld, scale)
    mo, _ = attention64(q, k, v, ld, scale, absolute=True)
    close(o, eo, bound(dtype, 3000, mo), "o")
    assert torch.equal(o, F.linear_attention(q, k, v, ld, return_state=True)[0])
    got = F.linear_attention_backward(go, q, k, v, ld)
    exp, maj = attention64(q, k, v, ld, scale, None, None, go), attention64(q, k, v, ld, scale, None, None, go, absolute=True)
    for n, a, e, m in zip(("dq", "dk", "dv"), got, exp, maj):
        close(a, e, bound(dtype, 3000, m, 2), n)
    F.check_operators()


@pytest.mark.parametrize("size", [1e-3, 1.0, 200.0])
def test_fp16_sizes(F, size):
    """Inputs far from 1 on either side: the powers of two that bring them into fp16's range cost no precision."""
    g = gen(33)
    q, k = (randn(g, 1, 500, 2, 64) * size).half(), (randn(g, 1, 500, 2, 64) * size).half()
    v = (randn(g, 1, 500, 2, 64) * min(1.0, 1 / size)).half()
    ld, scale = decays(2), 0.125
    o, s = F.linear_attention(q, k, v, ld, return_state=True)
    eo, es = attention64(q, k, v, ld, scale)
    mo, ms = attention64(q, k, v, ld, scale, absolute=True)
    close(o, eo, bound(torch.float16, 500, mo) + 2.0 ** -25, "o")  # 2^-25: half of fp16's smallest number
    close(s, es, state_bound(500, ms), "state")


def test_refusals_of_tensors(F):
    from lama_b200 import LamaError
    z = torch.zeros(1, 4, 2, 64, device="cuda", dtype=torch.bfloat16)
    ld = torch.zeros(2, device="cuda")
    st = torch.zeros(1, 2, 64, 64, device="cuda")
    x = torch.zeros(2, 3, 8, device="cuda")
    w = torch.ones(8, device="cuda")
    cases = [
        (lambda: F.linear_attention(z, z.half(), z, ld), "k has type"),
        (lambda: F.linear_attention(z.int(), z, z, ld), "has type"),
        (lambda: F.linear_attention(z[0], z, z, ld), "dimensions"),
        (lambda: F.linear_attention(z, z[:, :3], z, ld), "does not go with"),
        (lambda: F.linear_attention(z, z[..., :8], z, ld), "channels a head"),
        (lambda: F.linear_attention(z, z, z, torch.zeros(3, device="cuda")), "do not divide"),
        (lambda: F.linear_attention(z, z, z, ld.cpu()), "log_decay is on cpu"),
        (lambda: F.linear_attention(z, z, z, ld.clone().requires_grad_()), "no gradient"),
        (lambda: F.linear_attention(z, z, z, ld, initial_state=st[:, :1]), "initial_state has shape"),
        (lambda: F.linear_attention(z, z, z, ld, lengths=torch.zeros(1, device="cuda")), "lengths has type"),
        (lambda: F.linear_attention(z, z, z, ld, scale="a"), "not a number"),
        (lambda: F.linear_attention(torch.zeros(1, 4, 2, 129, device="cuda"), torch.zeros(1, 4, 2, 129, device="cuda"),
                                    torch.zeros(1, 4, 2, 64, device="cuda"), ld), "1..128"),
        (lambda: F.linear_attention_backward(z[:, :3], z, z, z, ld), "grad_o has shape"),
        (lambda: F.linear_attention_step(z[:, 0], z[:, 0], z[:, 0], ld, st[..., :32]), "state is not a contiguous"),
        (lambda: F.linear_attention_step(z[:, 0], z[:, 0], z[:, 0], ld, st, out_state=st[0]), "out_state has shape"),
        (lambda: F.linear_attention_step(z[:, 0], z[:, 0], z[:, 0], ld, st, slots=torch.zeros(2, device="cuda",
                                                                                         dtype=torch.int32)), "slots has shape"),
        (lambda: F.linear_attention_step(z[:, 0].expand(2, 2, 64), z[:, 0].expand(2, 2, 64), z[:, 0].expand(2, 2, 64), ld, st),
         "1 states for 2 rows"),
        (lambda: F.linear_attention_step(z[:, 0].clone().requires_grad_(), z[:, 0], z[:, 0], ld, st), "no gradient"),
        (lambda: F.gated_residual_norm(x, x[:1]), "y has shape"),
        (lambda: F.gated_residual_norm(x, x.half()), "y has type"),
        (lambda: F.gated_residual_norm(x, x, post_weight=w[:4]), "post_weight is not"),
        (lambda: F.gated_residual_norm(x, x, gate=x[:, :2]), "does not broadcast"),
        (lambda: F.gated_residual_norm(x, x, gate=x[:1]), "expand it"),
        (lambda: F.gated_residual_norm(x, x, gate=x.half()), "gate has type"),
        (lambda: F.gated_residual_norm(x, x, residual_scale=w[:3]), "residual_scale is not"),
        (lambda: F.gated_residual_norm(x, x, eps=-1), "eps"),
        (lambda: F.checkpoint_store(x.int()), "has type"),
        (lambda: F.checkpoint_restore(F.Checkpoint8(x.to(torch.int8), x, torch.float32)), "scales has shape"),
    ]
    for f, msg in cases:
        with pytest.raises(LamaError) as ex:
            f()
        assert ex.value.code == -1 and msg in ex.value.msg, (msg, ex.value.msg)
    _, _, saved = F.gated_residual_norm(x, x, pre_weight=w, save="full")
    with pytest.raises(LamaError):
        F.gated_residual_norm_backward(x[:1], None, saved)
    F.check_operators()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("dk,dv,T", [(8, 8, 130), (16, 40, 260), (72, 24, 300), (24, 120, 1), (104, 128, 700)])
def test_head_sizes_that_fill_no_tile(F, dtype, dk, dv, T):
    g = gen(41)
    q, k, v, go = (randn(g, 2, T, 3, d, dtype=dtype) for d in (dk, dk, dv, dv))
    ld, scale, s0 = decays(3), dk ** -0.5, randn(g, 2, 3, dk, dv)
    lengths = torch.tensor([T, max(1, T - 5)], device="cuda", dtype=torch.int32)
    o, s = F.linear_attention(q, k, v, ld, initial_state=s0, lengths=lengths, return_state=True)
    eo, es = attention64(q, k, v, ld, scale, s0, lengths)
    mo, ms = attention64(q, k, v, ld, scale, s0, lengths, absolute=True)
    close(o, eo, bound(dtype, T, mo) + 2.0 ** -25, "o")
    close(s, es, state_bound(T, ms), "state")
    got = F.linear_attention_backward(go, q, k, v, ld, initial_state=s0, lengths=lengths)
    exp = attention64(q, k, v, ld, scale, s0, lengths, go)
    maj = attention64(q, k, v, ld, scale, s0, lengths, go, absolute=True)
    for n, a, e, m in zip(("dq", "dk", "dv"), got, exp, maj):
        close(a, e, bound(dtype, T, m, 3) + 2.0 ** -25, n)
    close(got[3], exp[3], state_bound(T, maj[3]), "ds0")
    F.check_operators()


def test_operators_in_a_cuda_graph(F):
    """Captured after a first call (which sets the kernels up) and replayed on new contents of the same tensors."""
    g = gen(43)
    q, k, v = (randn(g, 1, 700, 2, 64, dtype=torch.bfloat16) for _ in range(3))
    x, y = randn(g, 700, 128, dtype=torch.bfloat16), randn(g, 700, 128, dtype=torch.bfloat16)
    w, ld = torch.ones(128, device="cuda"), decays(2)

    def work():
        o, s = F.linear_attention(q, k, v, ld, return_state=True)
        u, n, saved = F.gated_residual_norm(x, y, post_weight=w, pre_weight=w, save="int8")
        return (o, s, u, n, *F.linear_attention_backward(o, q, k, v, ld)[:3], F.gated_residual_norm_backward(u, n, saved).y)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        work()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = work()
    for t in (q, k, v, x, y):
        t.copy_(randn(g, *t.shape, dtype=t.dtype))
    graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(out, work()):
        assert torch.equal(a, b)


def test_calls_from_several_threads(F):
    """Each thread on its own stream, sizes apart, results as alone."""
    import threading
    sizes = [(1, 300, 2, 64), (2, 1500, 1, 128), (1, 4000, 3, 64), (3, 90, 2, 32)]
    ins = [[randn(gen(50 + i), *s, dtype=torch.bfloat16) for _ in range(3)] for i, s in enumerate(sizes)]
    alone = [F.linear_attention(*x, decays(x[0].shape[2])) for x in ins]
    torch.cuda.synchronize()
    got, bad = [None] * len(ins), []

    def go(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(20):
                    got[i] = F.linear_attention(*ins[i], decays(ins[i][0].shape[2]))
                torch.cuda.current_stream().synchronize()
        except Exception as e:  # noqa: BLE001
            bad.append(e)
    ts = [threading.Thread(target=go, args=(i,)) for i in range(len(ins))]
    for t in ts:
        t.start()
    for t in ts:
        t.join()
    assert not bad, bad
    for a, b in zip(got, alone):
        assert torch.equal(a, b)
