"""What is measured of the token-mixer operators of lama_b200.operators.

Three operators that make up a trainable token-mixer block over the latent plane:

* linear attention with a decay for each head: whole sequences, their gradients, single tokens;
* the norm after a block, its gate and residual scale, the residual sum and the norm before the next
  block in one pass, and the gradients;
* activation checkpoints in 8 bits, stored, restored, and read by the norms' backward pass.

Sequences are latent planes in raster order: 64x64 tokens for a 512x512 image, 75x75 for a 600x600
window, 128x128 for 1024x1024, 256x256 for 2048x2048; widths are the generator's 128, 384 and 512
channels, or generic.  `run` computes either the plain form (elementary torch operations in 32 bits)
or, where `own` is true, calls the framework.
"""

import math
import os
import sys

import torch

own = False

GROUP = 128         # channels that share one scale of an 8-bit checkpoint
TINY = 2.0 ** -96   # a group whose largest magnitude is below this is stored as zeros
EPS = 1e-6

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ------------------------------------------------------------------ cases

def _la(name, op, dtype, b, t, h, dk, dv, hq=None, hk=None, hv=None, ragged=False, state=False):
    return {"name": name, "op": op, "dtype": dtype, "b": b, "t": t, "h": h, "dk": dk, "dv": dv, "hq": hq or h,
            "hk": hk or h, "hv": hv or h, "ragged": ragged, "state": state}


def _step(name, dtype, b, h, dk, dv, hq=None, hk=None, hv=None, slots=False):
    return {"name": name, "op": "step", "dtype": dtype, "b": b, "h": h, "dk": dk, "dv": dv, "hq": hq or h,
            "hk": hk or h, "hv": hv or h, "slots": slots}


def _norm(name, op, dtype, b, t, c, gate, save="full"):
    return {"name": name, "op": op, "dtype": dtype, "b": b, "t": t, "c": c, "gate": gate, "save": save}


def listed():
    return [
        # a 512x512 image's latent through one layer, the state kept for what follows
        _la("prompt_512", "prompt", "bf16", 1, 4096, 8, 64, 64, state=True),
        # two 600x600 windows cut to their hole, so of different lengths; the keys and queries shared by heads
        _la("prompt_window_ragged", "prompt", "fp16", 2, 5625, 6, 64, 80, hq=3, hk=3, ragged=True, state=True),
        # 2048x2048 images in batch
        _la("prompt_2048", "prompt", "bf16", 2, 65536, 4, 128, 128),
        # fine-tuning in mixed precision on 512x512 images: output and gradients
        _la("train_512", "train", "bf16", 16, 4096, 8, 64, 64),
        # a small full-precision step on 312x312 crops (39x39 tokens), values shared by heads
        _la("train_crop_fp32", "train", "fp32", 2, 1521, 4, 64, 64, hv=2, state=True),
        # one stream, one token: latency
        _step("step_one", "bf16", 1, 8, 64, 64),
        # a server's streams, their states in a pool of slots, some rows of the batch unused
        _step("step_pool", "bf16", 256, 8, 128, 128, slots=True),
        # the glue of one block at inference, a gate for each image
        _norm("norm_512", "norm", "bf16", 1, 4096, 512, "image"),
        # a training step with 8-bit checkpoints on a batch of 512x512 images
        _norm("norm_train_int8", "norm_train", "bf16", 32, 4096, 512, "image", save="int8"),
        # a full-precision training step on 600x600 windows, a gate for each token and channel
        _norm("norm_train_window", "norm_train", "fp32", 2, 5625, 384, "token"),
        # one activation of a 16-image batch stored and restored
        {"name": "store_512", "op": "store", "dtype": "bf16", "rows": 16 * 4096, "c": 512},
        # a small odd one in full precision: its last group is ragged
        {"name": "store_odd", "op": "store", "dtype": "fp32", "rows": 1521, "c": 397},
    ]


def _log_int(rng, lo, hi):
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    return 3071 if v == 3072 else max(lo, min(hi, v))


def draw(rng):
    most = {}
    for c in listed():
        w = work(c)
        kind = c["op"].split("_")[0]
        most[kind] = max(most.get(kind, 0), w["bytes"])
    while True:
        op = rng.choice(["prompt", "prompt", "train", "train", "step", "norm", "norm_train", "store"])
        dtype = rng.choice(["bf16", "bf16", "bf16", "fp16", "fp32"])
        if op in ("prompt", "train", "step"):
            h = rng.choice([1, 2, 3, 4, 6, 8, 16])
            div = [d for d in range(1, h + 1) if h % d == 0]
            heads = {n: h if rng.random() < 0.6 else rng.choice(div) for n in ("hq", "hk", "hv")}
            dk = rng.choice([16, 33, 64, 64, 64, 80, 128, 128])
            dv = dk if rng.random() < 0.6 else rng.choice([16, 33, 64, 64, 80, 128])
            if op == "step":
                case = _step(None, dtype, _log_int(rng, 1, 512), h, dk, dv, slots=rng.random() < 0.5, **heads)
            else:
                case = _la(None, op, dtype, _log_int(rng, 1, 16), _log_int(rng, 16, 65536), h, dk, dv,
                           ragged=rng.random() < 0.3, state=rng.random() < 0.5, **heads)
        elif op in ("norm", "norm_train"):
            c = rng.choice([128, 384, 512, 512, 257, 1000, 1024, 2048, _log_int(rng, 64, 8192)])
            case = _norm(None, op, dtype, _log_int(rng, 1, 32), _log_int(rng, 1, 65536), c,
                         rng.choice(["none", "image", "token"]), rng.choice(["full", "int8"]))
        else:
            case = {"op": op, "dtype": dtype, "rows": _log_int(rng, 1, 131072),
                    "c": rng.choice([128, 384, 512, 397, _log_int(rng, 16, 8192)])}
        case.pop("name", None)
        if work(case)["bytes"] <= most[op.split("_")[0]]:
            return case


# ------------------------------------------------------------------ inputs

def _lengths(case, gen):
    return torch.randint(0, case["t"] + 1, (case["b"],), generator=gen, device="cuda", dtype=torch.int32)


def _log_decay(h):
    # fixed slopes from half a token to some thousand tokens of memory, one for each head
    return torch.tensor([-math.exp(math.log(0.7) + (math.log(3e-4) - math.log(0.7)) * i / max(h - 1, 1))
                         for i in range(h)], dtype=torch.float32, device="cuda")


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    dt = TYPES[case["dtype"]]

    def randn(*shape, dtype=dt, scale=1.0):
        return (torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32) * scale).to(dtype)

    op = case["op"]
    st = {"case": case, "op": op}
    if op in ("prompt", "train"):
        b, t, dk, dv = case["b"], case["t"], case["dk"], case["dv"]
        st.update(q=randn(b, t, case["hq"], dk), k=randn(b, t, case["hk"], dk), v=randn(b, t, case["hv"], dv),
                  g=_log_decay(case["h"]), scale=dk ** -0.5, s0=None, lengths=None)
        if case["state"]:
            st["s0"] = randn(b, case["h"], dk, dv, dtype=torch.float32, scale=2.0)
        if case["ragged"]:
            st["lengths"] = _lengths(case, gen)
        if op == "train":
            st["go"] = randn(b, t, case["h"], dv)
    elif op == "step":
        b, h, dk, dv = case["b"], case["h"], case["dk"], case["dv"]
        n = b + b // 4 if case["slots"] else b
        st.update(q=randn(b, case["hq"], dk), k=randn(b, case["hk"], dk), v=randn(b, case["hv"], dv),
                  g=_log_decay(h), scale=dk ** -0.5,
                  state=randn(n, h, dk, dv, dtype=torch.float32, scale=4.0), slots=None)
        st["out_state"] = st["state"].clone()
        if case["slots"]:
            s = torch.randperm(n, generator=gen, device="cuda")[:b].to(torch.int32)
            unused = torch.rand(b, generator=gen, device="cuda") < 0.1
            st["slots"] = torch.where(unused, torch.full_like(s, -1), s)
    elif op in ("norm", "norm_train"):
        b, t, c = case["b"], case["t"], case["c"]
        # a residual stream has a few channels far larger than the rest
        chan = torch.exp(torch.randn(c, generator=gen, device="cuda") * 0.7)
        st.update(x=(randn(b, t, c, dtype=torch.float32) * chan * 2).to(dt), y=randn(b, t, c, scale=0.5),
                  w_post=1 + randn(c, dtype=torch.float32, scale=0.2),
                  w_pre=1 + randn(c, dtype=torch.float32, scale=0.2),
                  s=0.5 + randn(c, dtype=torch.float32, scale=0.1), gate=None)
        if case["gate"] != "none":
            st["gate"] = randn(b, 1 if case["gate"] == "image" else t, c, scale=0.7)
        if op == "norm_train":
            st["gu"], st["gn"] = randn(b, t, c), randn(b, t, c)
    else:
        chan = torch.exp(torch.randn(case["c"], generator=gen, device="cuda") * 0.7)
        st["x"] = (randn(case["rows"], case["c"], dtype=torch.float32) * chan).to(dt)
    return st


# ------------------------------------------------------------------ one pass

def _framework():
    package = os.path.join(os.getcwd(), "lama-inpaint-rs_b200")
    if package not in sys.path:
        sys.path.insert(1, package)
    from lama_b200 import operators
    return operators


def run(st):
    op = st["op"]
    if own:
        F = _framework()
        if op == "prompt":
            return F.linear_attention(st["q"], st["k"], st["v"], st["g"], scale=st["scale"],
                                      initial_state=st["s0"], lengths=st["lengths"], return_state=True)
        if op == "train":
            kw = dict(scale=st["scale"], initial_state=st["s0"], lengths=st["lengths"])
            o = F.linear_attention(st["q"], st["k"], st["v"], st["g"], **kw)
            dq, dk, dv, ds0 = F.linear_attention_backward(st["go"], st["q"], st["k"], st["v"], st["g"], **kw)
            return (o, dq, dk, dv) if ds0 is None else (o, dq, dk, dv, ds0)
        if op == "step":
            o = F.linear_attention_step(st["q"], st["k"], st["v"], st["g"], st["state"], scale=st["scale"],
                                        slots=st["slots"], out_state=st["out_state"])
            return o, st["out_state"]
        if op == "norm":
            return F.gated_residual_norm(st["x"], st["y"], post_weight=st["w_post"], pre_weight=st["w_pre"],
                                         gate=st["gate"], residual_scale=st["s"], eps=EPS)
        if op == "norm_train":
            u, n, saved = F.gated_residual_norm(st["x"], st["y"], post_weight=st["w_post"], pre_weight=st["w_pre"],
                                                gate=st["gate"], residual_scale=st["s"], eps=EPS,
                                                save=st["case"]["save"])
            gr = F.gated_residual_norm_backward(st["gu"], st["gn"], saved)
            out = [u, n, gr.x, gr.y, gr.post_weight, gr.pre_weight, gr.residual_scale]
            return out if st["gate"] is None else out + [gr.gate]
        return F.checkpoint_restore(F.checkpoint_store(st["x"]))
    if op == "prompt":
        return _plain_forward(st)
    if op == "train":
        o, _ = _plain_forward(st)
        grads = _plain_backward(st)
        return (o,) + (grads if st["s0"] is not None else grads[:3])
    if op == "step":
        return _plain_step(st)
    if op == "norm":
        return _plain_norm(st)[:2]
    if op == "norm_train":
        return _plain_norm_train(st)
    codes, scale = _plain_codes(st["x"].float())
    return _plain_values(codes, scale, st["x"].shape[-1]).to(st["x"].dtype)


# ------------------------------------------------------------------ plain forms

CHUNK = 128


def _power(g, n):
    """exp(g)^n for n >= 0, and 1 for n = 0 whatever g is."""
    n = n.float()
    return torch.where(n == 0, torch.ones_like(n * g), torch.exp(g * n))


def _heads(x, h):
    """[B,T,n,D] to [B,H,T,D] in 32 bits, each of the n heads repeated for the H/n that share it."""
    return x.float().repeat_interleave(h // x.shape[2], 2).transpose(1, 2)


def _chunks(st):
    """Per chunk: first token, its number of tokens, how many of them each sequence has [B,1,1,1]."""
    b, t = st["q"].shape[:2]
    dev = st["q"].device
    lens = st["lengths"] if st["lengths"] is not None else torch.full((b,), t, device=dev)
    for c0 in range(0, t, CHUNK):
        c = min(CHUNK, t - c0)
        yield c0, c, (lens - c0).clamp(0, c).view(b, 1, 1, 1)


def _plain_states(st, q, k, v, g):
    b, h = q.shape[:2]
    s = st["s0"].float() if st["s0"] is not None else q.new_zeros(b, h, k.shape[-1], v.shape[-1])
    states = []
    for c0, c, n in _chunks(st):
        states.append(s)
        j = torch.arange(c, device=q.device).view(1, 1, c, 1)
        w = torch.where(j < n, _power(g, (n - 1 - j).clamp_min(0)), 0.0)
        s = _power(g, n) * s + (k[:, :, c0:c0 + c] * w).transpose(-1, -2) @ v[:, :, c0:c0 + c]
    return states, s


def _plain_forward(st):
    h = st["g"].numel()
    q, k, v = (_heads(st[n], h) for n in "qkv")
    g = st["g"].view(1, h, 1, 1)
    states, last = _plain_states(st, q, k, v, g)
    o = torch.empty(*q.shape[:3], v.shape[-1], device=q.device)
    for (c0, c, n), s in zip(_chunks(st), states):
        i = torch.arange(c, device=q.device).view(1, 1, c, 1)
        d = i - i.transpose(-1, -2)
        qc = q[:, :, c0:c0 + c] * (i < n)
        a = (qc @ k[:, :, c0:c0 + c].transpose(-1, -2)) * torch.where(d >= 0, _power(g, d.clamp_min(0)), 0.0)
        o[:, :, c0:c0 + c] = a @ v[:, :, c0:c0 + c] + (qc * _power(g, i + 1)) @ s
    return (o * st["scale"]).transpose(1, 2).to(st["q"].dtype).contiguous(), last


def _plain_backward(st):
    h = st["g"].numel()
    q, k, v = (_heads(st[n], h) for n in "qkv")
    go = st["go"].float().transpose(1, 2) * st["scale"]
    g = st["g"].view(1, h, 1, 1)
    states, last = _plain_states(st, q, k, v, g)
    ds = torch.zeros_like(last)
    dq, dk, dv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
    for (c0, c, n), s in reversed(list(zip(_chunks(st), states))):
        i = torch.arange(c, device=q.device).view(1, 1, c, 1)
        on = i < n
        d = i - i.transpose(-1, -2)
        decay = torch.where(d >= 0, _power(g, d.clamp_min(0)), 0.0)
        sl = slice(c0, c0 + c)
        qc, kc, vc, gc = q[:, :, sl] * on, k[:, :, sl] * on, v[:, :, sl] * on, go[:, :, sl] * on
        a = (qc @ kc.transpose(-1, -2)) * decay
        p = (gc @ vc.transpose(-1, -2)) * decay
        w_in = _power(g, i + 1)
        w_out = torch.where(on, _power(g, (n - 1 - i).clamp_min(0)), 0.0)
        dq[:, :, sl] = p @ kc + (gc * w_in) @ s.transpose(-1, -2)
        dk[:, :, sl] = p.transpose(-1, -2) @ qc + (vc * w_out) @ ds.transpose(-1, -2)
        dv[:, :, sl] = a.transpose(-1, -2) @ gc + (kc * w_out) @ ds
        ds = _power(g, n) * ds + (qc * w_in).transpose(-1, -2) @ gc

    def back(x, like):
        b, _, t, d = x.shape
        n = like.shape[2]
        return x.transpose(1, 2).reshape(b, t, n, h // n, d).sum(3).to(like.dtype)

    return back(dq, st["q"]), back(dk, st["k"]), back(dv, st["v"]), ds


def _plain_step(st):
    h = st["g"].numel()
    q, k, v = (st[n].float().repeat_interleave(h // st[n].shape[1], 1) for n in "qkv")
    lam = torch.exp(st["g"]).view(1, h, 1, 1)
    slots = st["slots"]
    if slots is None:
        s = lam * st["state"] + k[..., :, None] * v[..., None, :]
        o = (q[..., :, None] * s).sum(2) * st["scale"]
        st["out_state"].copy_(s)
        return o.to(st["q"].dtype), st["out_state"]
    used = slots >= 0
    at = torch.where(used, slots, 0).long()
    s = lam * st["state"][at] + k[..., :, None] * v[..., None, :]
    o = (q[..., :, None] * s).sum(2) * st["scale"] * used.view(-1, 1, 1)
    st["out_state"][at[used]] = s[used]
    return o.to(st["q"].dtype), st["out_state"]


def _plain_norm(st):
    x, y = st["x"].float(), st["y"].float()
    ry = torch.rsqrt((y * y).mean(-1, keepdim=True) + EPS)
    p = y * ry * st["w_post"]
    gate = 1.0 if st["gate"] is None else st["gate"].float()
    u = (x + st["s"] * gate * p).to(st["x"].dtype)  # the stream carries the rounded sum
    uf = u.float()
    ru = torch.rsqrt((uf * uf).mean(-1, keepdim=True) + EPS)
    return u, (uf * ru * st["w_pre"]).to(u.dtype), ry, ru


def _plain_codes(x):
    c = x.shape[-1]
    groups = (c + GROUP - 1) // GROUP
    x = torch.nn.functional.pad(x, (0, groups * GROUP - c)).view(*x.shape[:-1], groups, GROUP)
    a = x.abs().amax(-1, keepdim=True)
    top = torch.full_like(a, 127.0)  # a tensor: torch divides by a number through its reciprocal, in two roundings
    inv = torch.where(a < TINY, 0.0, top / a)
    return torch.round(x * inv).to(torch.int8), torch.where(a < TINY, 0.0, a / top)


def _plain_values(codes, scale, c):
    return (codes.float() * scale).flatten(-2)[..., :c]


def _plain_norm_train(st):
    u, n, ry, ru = _plain_norm(st)
    y, uh = st["y"].float(), u.float()
    if st["case"]["save"] == "int8":
        y = _plain_values(*_plain_codes(y), y.shape[-1])
        uh = _plain_values(*_plain_codes(uh), uh.shape[-1])
    gu, gn = st["gu"].float(), st["gn"].float()
    gate = 1.0 if st["gate"] is None else st["gate"].float()
    wn = gn * st["w_pre"]
    uh = uh * ru
    du = gu + ru * (wn - uh * (uh * wn).mean(-1, keepdim=True))
    yh = y * ry
    dp = du * st["s"] * gate
    wp = dp * st["w_post"]
    dy = ry * (wp - yh * (yh * wp).mean(-1, keepdim=True))
    rows = (0, 1)
    out = [u, n, du.to(u.dtype), dy.to(u.dtype), (dp * yh).sum(rows), (gn * uh).sum(rows),
           (du * gate * yh * st["w_post"]).sum(rows)]
    if st["gate"] is not None:
        dg = du * st["s"] * yh * st["w_post"]
        out.append((dg.sum(1, keepdim=True) if st["case"]["gate"] == "image" else dg).to(u.dtype))
    return out


# ------------------------------------------------------------------ 64 bits

def exact(case, seed):
    st = prepare(case, seed)
    op = case["op"]
    if op in ("prompt", "train"):
        return _exact_attention(case, st)
    if op == "step":
        return _exact_step(st)
    if op in ("norm", "norm_train"):
        return _exact_norm(case, st)
    return None  # what 8 bits hold is compared with the plain form, value for value


def _exact_attention(case, st):
    """The sums over all earlier tokens written out, a block of rows at a time."""
    b, t, h = case["b"], case["t"], case["h"]
    train = case["op"] == "train"
    out = {n: torch.zeros(*st[n].shape, dtype=torch.float64, device="cuda") for n in "qkv"}
    o = torch.zeros(b, t, h, case["dv"], dtype=torch.float64, device="cuda")
    last = torch.zeros(b, h, case["dk"], case["dv"], dtype=torch.float64, device="cuda")
    ds0 = torch.zeros_like(last)
    lens = [t] * b if st["lengths"] is None else st["lengths"].tolist()
    for bi in range(b):
        for hi in range(h):
            n = lens[bi]
            at = {x: hi // (h // case["h" + x]) for x in "qkv"}
            q, k, v = (st[x][bi, :n, at[x]].double() for x in "qkv")
            g = st["g"][hi].double()
            s0 = None if st["s0"] is None else st["s0"][bi, hi].double()
            do = st["go"][bi, :n, hi].double() * st["scale"] if train else None
            pos = torch.arange(n, device="cuda", dtype=torch.float64)
            for r0 in range(0, n, 2048):
                r1 = min(n, r0 + 2048)
                dist = pos[r0:r1, None] - pos[None, :r1]
                m = torch.exp(g * dist.clamp_min(0)) * (dist >= 0)
                a = (q[r0:r1] @ k[:r1].T) * m
                o[bi, r0:r1, hi] = a @ v[:r1]
                w = torch.exp(g * (pos[r0:r1, None] + 1))
                if s0 is not None:
                    o[bi, r0:r1, hi] += w * (q[r0:r1] @ s0)
                if train:
                    d = do[r0:r1]
                    p = (d @ v[:r1].T) * m
                    out["q"][bi, r0:r1, at["q"]] += p @ k[:r1]
                    out["k"][bi, :r1, at["k"]] += p.T @ q[r0:r1]
                    out["v"][bi, :r1, at["v"]] += a.T @ d
                    if s0 is not None:
                        out["q"][bi, r0:r1, at["q"]] += w * (d @ s0.T)
                    ds0[bi, hi] += (q[r0:r1] * w).T @ d
            last[bi, hi] = (k * torch.exp(g * (n - 1 - pos[:, None]))).T @ v
            if s0 is not None:
                last[bi, hi] += torch.exp(g * n) * s0
    o *= st["scale"]
    if not train:
        return o, last
    res = (o, out["q"], out["k"], out["v"])
    return res + (ds0,) if st["s0"] is not None else res


def _exact_step(st):
    h = st["g"].numel()
    o = torch.zeros(st["q"].shape[0], h, st["v"].shape[-1], dtype=torch.float64, device="cuda")
    state = st["state"].double()
    rows = range(o.shape[0])
    slots = list(rows) if st["slots"] is None else st["slots"].tolist()
    lam = torch.exp(st["g"].double()).view(h, 1, 1)
    idx = {n: torch.arange(h, device="cuda") // (h // st[n].shape[1]) for n in "qkv"}
    for r in rows:
        if slots[r] < 0:
            continue
        q, k, v = (st[n][r].double()[idx[n]] for n in "qkv")
        state[slots[r]] = lam * state[slots[r]] + torch.einsum("hk,hv->hkv", k, v)
        o[r] = torch.einsum("hk,hkv->hv", q, state[slots[r]]) * st["scale"]
    return o, state


def _exact_codes(x):
    c = x.shape[-1]
    v = x.clone()
    for c0 in range(0, c, GROUP):
        part = v[..., c0:c0 + GROUP]
        step = part.abs().amax(-1, keepdim=True) / 127
        part.copy_(torch.where(step > 0, torch.round(part / step.clamp_min(1e-300)) * step, 0.0))
    return v


def _exact_norm(case, st):
    f = {n: (None if st[n] is None else st[n].double()) for n in ("x", "y", "w_post", "w_pre", "s", "gate")}
    train = case["op"] == "norm_train"
    parts = []
    sums = None
    for bi in range(case["b"]):  # one image at a time: 64 bits of the largest batch would be many GB
        x, y = f["x"][bi], f["y"][bi]
        gate = torch.ones((), dtype=torch.float64, device="cuda") if f["gate"] is None else f["gate"][bi]
        ny = 1 / torch.sqrt(torch.mean(y ** 2, -1, keepdim=True) + EPS)
        u = x + f["s"] * gate * f["w_post"] * y * ny
        nu = 1 / torch.sqrt(torch.mean(u ** 2, -1, keepdim=True) + EPS)
        row = [u, f["w_pre"] * u * nu]
        if train:
            yk, uk = (_exact_codes(y), _exact_codes(u)) if case["save"] == "int8" else (y, u)
            gu, gn = st["gu"][bi].double(), st["gn"][bi].double()
            back = f["w_pre"] * gn
            dx = gu + nu * back - uk * nu ** 3 * torch.mean(uk * back, -1, keepdim=True)
            dp = dx * f["s"] * gate
            back = f["w_post"] * dp
            row += [dx, ny * back - yk * ny ** 3 * torch.mean(yk * back, -1, keepdim=True)]
            new = [(dp * yk * ny).sum(0), (gn * uk * nu).sum(0), (dx * gate * f["w_post"] * yk * ny).sum(0)]
            sums = new if sums is None else [p + q for p, q in zip(sums, new)]
            if f["gate"] is not None:
                dg = dx * f["s"] * f["w_post"] * yk * ny
                row.append(dg.sum(0, keepdim=True) if case["gate"] == "image" else dg)
        parts.append(row)
    out = [torch.stack(p) for p in zip(*parts)]
    return out if not train else out[:4] + sums + out[4:]


# ------------------------------------------------------------------ work

def work(case):
    op = case["op"]
    e = {"bf16": 2, "fp16": 2, "fp32": 4}[case["dtype"]]
    if op in ("prompt", "train"):
        b, t, h, dk, dv = case["b"], case["t"], case["h"], case["dk"], case["dv"]
        tokens = b * t
        inputs = (case["hq"] + case["hk"]) * dk + case["hv"] * dv
        state = 4 * b * h * dk * dv
        if op == "prompt":
            # q, k, v and the first state read, o and the last state written; 2 products a token and head
            return {"bytes": tokens * e * (inputs + h * dv) + state * (1 + case["state"]),
                    "flops": 4 * tokens * h * dk * dv}
        # q, k, v, do read, o, dq, dk, dv written; 2 products forward and 5 backward
        return {"bytes": tokens * e * 2 * (inputs + h * dv) + 2 * state * case["state"],
                "flops": 14 * tokens * h * dk * dv}
    if op == "step":
        b, h, dk, dv = case["b"], case["h"], case["dk"], case["dv"]
        return {"bytes": 8 * b * h * dk * dv + b * e * ((case["hq"] + case["hk"]) * dk + (case["hv"] + h) * dv),
                "flops": 5 * b * h * dk * dv}
    if op in ("norm", "norm_train"):
        rows, c = case["b"] * case["t"], case["c"]
        gate = {"none": 0, "image": case["b"] * c, "token": rows * c}[case["gate"]]
        if op == "norm":
            return {"bytes": e * (4 * rows * c + gate) + 12 * c, "flops": 11 * rows * c}
        # x, y, du, dn and the gate read; u, n, dx, dy, the gate's gradient and three vectors written
        return {"bytes": e * (8 * rows * c + 2 * gate) + 24 * c, "flops": 40 * rows * c}
    # read, stored as codes and scales, read back, written
    n = case["rows"] * case["c"]
    scales = 4 * case["rows"] * ((case["c"] + GROUP - 1) // GROUP)
    return {"bytes": 2 * n * e + 2 * (n + scales), "flops": 4 * n}
