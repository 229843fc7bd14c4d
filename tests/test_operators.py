"""Refusals of the token-mixer operators, without a GPU: the C ABI checks sizes, types, strides and pointers
before any CUDA call, and the torch binding checks tensors before it calls the library."""

import ctypes
import struct

import pytest
import torch

from lama_b200 import LamaError
from lama_b200 import engine as E

EINVAL, EUNSUPPORTED = -1, -6


def rows(data=4096, heads=2):
    return struct.pack("@Pqqqi4x", data, 64, 64, 64, heads)


def attention(dtype=2, batch=1, tokens=10, heads=2, dk=64, dv=64, q=None, k=None, v=None, decay=4096, init=0, lengths=0):
    return struct.pack("@6i", dtype, batch, tokens, heads, dk, dv) + (q or rows()) + (k or rows()) + (v or rows()) + \
        struct.pack("@3Pf4x", decay, init, lengths, 1.0)


def call(name, *args):
    err = ctypes.create_string_buffer(256)
    rc = getattr(E.lib(), name)(*args, err, 256)
    return rc, err.value.decode()


@pytest.mark.parametrize("kw,code,msg", [
    (dict(dtype=3), EINVAL, "element type"), (dict(batch=0), EINVAL, "must be positive"),
    (dict(tokens=0), EINVAL, "must be positive"), (dict(dk=129), EUNSUPPORTED, "exceed 128"),
    (dict(dv=200), EUNSUPPORTED, "exceed 128"), (dict(decay=0), EINVAL, "log_decay is null"),
    (dict(q=rows(0)), EINVAL, "q is null"), (dict(k=rows(4097)), EINVAL, "k is not aligned"),
    (dict(v=rows(heads=3)), EINVAL, "v has 3 heads"), (dict(batch=40000), EUNSUPPORTED, "65535"),
])
def test_attention_refuses(kw, code, msg):
    rc, text = call("lama_linear_attention_workspace", attention(**kw), 0)
    assert rc == code and msg in text
    rc, text = call("lama_linear_attention", attention(**kw), rows(), None, None, 0, 0, None)
    assert rc == code and msg in text


def test_attention_refuses_bad_outputs_and_workspaces():
    a = attention(tokens=4096, batch=1)
    need, _ = call("lama_linear_attention_workspace", a, 0)
    assert need > 0
    rc, text = call("lama_linear_attention", a, rows(), None, None, 0, 0, None)
    assert rc == EINVAL and f"{need} needed" in text
    rc, text = call("lama_linear_attention", a, rows(heads=1), None, 4096, need, 0, None)
    assert rc == EINVAL and "out has 1 heads" in text
    rc, text = call("lama_linear_attention", a, None, None, 4096, need, 0, None)
    assert rc == EINVAL
    assert call("lama_linear_attention", None, rows(), None, None, 0, 0, None)[0] == EINVAL
    need, _ = call("lama_linear_attention_workspace", a, 1)
    g = rows() * 4 + struct.pack("@2P", 0, 0)
    rc, text = call("lama_linear_attention_backward", a, g, None, 0, 0, None)
    assert rc == EINVAL and "needed" in text
    bad = rows() + rows(heads=1) + rows() * 2 + struct.pack("@2P", 0, 0)
    rc, text = call("lama_linear_attention_backward", a, bad, 4096, need, 0, None)
    assert rc == EINVAL and "grad_q has 1 heads" in text


@pytest.mark.parametrize("kw,args,msg", [
    (dict(tokens=2), (4096, 4096, 4, None), "one token"), (dict(tokens=1, lengths=4096), (4096, 4096, 4, None), "no lengths"),
    (dict(tokens=1, batch=5), (4096, 4096, 4, None), "4 slots for 5 rows"), (dict(tokens=1), (None, 4096, 4, None), "null"),
    (dict(tokens=1), (4096, 4096, 0, None), "must be positive"), (dict(tokens=1, q=rows(heads=3)), (4096, 4096, 4, None), "q has 3"),
])
def test_step_refuses(kw, args, msg):
    rc, text = call("lama_linear_attention_step", attention(**kw), rows(), *args, 0, None)
    assert rc == EINVAL and msg in text


def norm(dtype=2, n=4, c=64, gate=0, per=1, stride=64, post=4096, pre=4096, scales=0, scale=1.0, eps=1e-6):
    return struct.pack("@i4xqi4xPqq3P2f", dtype, n, c, gate, per, stride, post, pre, scales, scale, eps)


@pytest.mark.parametrize("kw,code,msg", [
    (dict(dtype=-1), EINVAL, "element type"), (dict(n=0), EINVAL, "must be positive"),
    (dict(c=16385), EUNSUPPORTED, "exceed 16384"), (dict(n=1 << 40), EUNSUPPORTED, "rows exceed"),
    (dict(gate=4096, per=0), EINVAL, "gate_rows"), (dict(eps=-1.0), EINVAL, "eps"), (dict(eps=float("nan")), EINVAL, "eps"),
])
def test_norm_refuses(kw, code, msg):
    rc, text = call("lama_gated_residual_norm_workspace", norm(**kw))
    assert rc == code and msg in text
    p = 4096
    rc, text = call("lama_gated_residual_norm", norm(**kw), p, 64, p, 64, p, p, None, None, None, None, None, None, 0, None)
    assert rc == code and msg in text


def test_norm_refuses_missing_tensors():
    p = 4096
    none = (None,) * 6
    for args, msg in (((None, 64, p, 64, p, p), "null"), ((p, 64, p, 64, p, None), "null"),
                      ((p, 63, p, 64, p, p), "row stride")):
        rc, text = call("lama_gated_residual_norm", norm(), *args, *none, 0, None)
        assert rc == EINVAL and msg in text
    rc, text = call("lama_gated_residual_norm", norm(), p, 64, p, 64, p, p, None, None, p, None, None, None, 0, None)
    assert rc == EINVAL and "codes without scales" in text
    need, _ = call("lama_gated_residual_norm_workspace", norm())

    def grads(gu=p, gn=p, y=p, u=p, strides=(64,) * 4, yc=0, uc=0, ys=0, us=0, ry=p, ru=p, gx=p, gy=p):
        return struct.pack("@4P4q12P", gu, gn, y, u, *strides, yc, uc, ys, us, ry, ru, gx, gy, 0, 0, 0, 0)
    for g, msg in ((grads(gx=0), "grad_x"), (grads(y=0), "neither y"), (grads(u=0), "neither u"),
                   (grads(ry=0), "statistics"), (grads(yc=p), "neither y"), (grads(strides=(64, 64, 10, 64)), "row stride")):
        rc, text = call("lama_gated_residual_norm_backward", norm(), g, p, need, 0, None)
        assert rc == EINVAL and msg in text, msg
    rc, text = call("lama_gated_residual_norm_backward", norm(), grads(), p, need - 1, 0, None)
    assert rc == EINVAL and f"{need} needed" in text


@pytest.mark.parametrize("args,msg", [
    ((None, 2, 4, 64, 64, 4096, 4096), "null"), ((4096, 9, 4, 64, 64, 4096, 4096), "element type"),
    ((4096, 2, 0, 64, 64, 4096, 4096), "must be positive"), ((4096, 2, 4, 64, 63, 4096, 4096), "row stride"),
    ((4097, 2, 4, 64, 64, 4096, 4096), "not aligned"),
])
def test_checkpoint_refuses(args, msg):
    rc, text = call("lama_checkpoint_store", *args, 0, None)
    assert rc == EINVAL and msg in text
    x, dtype, n, c, stride, codes, scales = args
    rc, text = call("lama_checkpoint_restore", codes, scales, dtype, n, c, stride, x, 0, None)
    assert rc == EINVAL and msg in text


def test_binding_refuses_tensors_of_the_host_and_other_objects():
    from lama_b200 import operators as F
    t = torch.zeros(1, 4, 2, 64)
    for f in (lambda: F.linear_attention(t, t, t, torch.zeros(2)), lambda: F.linear_attention(1, t, t, t),
              lambda: F.linear_attention_step(t[0], t[0], t[0], torch.zeros(2), t), lambda: F.checkpoint_store(t),
              lambda: F.checkpoint_store(None), lambda: F.gated_residual_norm(t, t),
              lambda: F.gated_residual_norm(t, t, save="half"), lambda: F.checkpoint_restore(t),
              lambda: F.linear_attention_backward(t, t, t, t, torch.zeros(2))):
        with pytest.raises(LamaError) as ex:
            f()
        assert ex.value.code == EINVAL
