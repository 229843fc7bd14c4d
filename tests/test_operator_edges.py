"""What the token-mixer operators refuse or pass on before any GPU is involved: autograd's demands on the
Python side, pointers and sizes at the C ABI."""

import struct

import pytest
import torch

from lama_b200 import LamaError

EINVAL = -1


def refused(f, msg):
    with pytest.raises(LamaError) as ex:
        f()
    assert ex.value.code == EINVAL and msg in ex.value.msg, ex.value.msg


# ------------------------------------------------------------------ autograd

def test_decays_that_want_a_gradient_are_refused_in_training_too():
    """They are constants: a gradient of None would leave a learnable decay as it is without a word."""
    from lama_b200 import operators as F
    z = torch.zeros(1, 4, 2, 8)
    s = torch.zeros(1, 2, 8, 8)
    ld = torch.zeros(2, requires_grad=True)
    for kw in (dict(q=1), dict(k=1), dict(v=1), dict(initial_state=1), dict(q=1, k=1, v=1)):
        t = {n: (s if n == "initial_state" else z).clone().requires_grad_() for n in kw}
        refused(lambda: F.linear_attention(t.get("q", z), t.get("k", z), t.get("v", z), ld,
                                           initial_state=t.get("initial_state")), "log_decay has no gradient")


def test_forward_mode_tangents_are_refused():
    """The kernels have no forward-mode form; results without the tangent would be derivatives of zero."""
    from lama_b200 import operators as F
    z, ld = torch.randn(1, 4, 2, 8), torch.zeros(2)
    with torch.autograd.forward_ad.dual_level():
        d = torch.autograd.forward_ad.make_dual(z, torch.ones_like(z))
        refused(lambda: F.linear_attention(d, z, z, ld), "forward-mode")
        refused(lambda: F.linear_attention(d[:, :, :1], z, z, ld), "forward-mode")  # a view has its base's
        refused(lambda: F.linear_attention_step(d[:, 0], z[:, 0], z[:, 0], ld, torch.zeros(1, 2, 8, 8)), "forward-mode")
        refused(lambda: F.gated_residual_norm(d, z, save="int8"), "forward-mode")
        refused(lambda: F.checkpoint_store(d), "forward-mode")
    refused(lambda: F.linear_attention(z, z, z, ld), "not on a CUDA device")  # plain tensors reach the next check


def test_a_checkpoint_of_a_tensor_that_wants_a_gradient_is_refused():
    """Codes have no gradient: taken from a graph they would cut it without a word."""
    from lama_b200 import operators as F
    x = torch.zeros(2, 8, requires_grad=True)
    refused(lambda: F.checkpoint_store(x), "has no gradient")
    with torch.no_grad():
        refused(lambda: F.checkpoint_store(x), "not on a CUDA device")
    refused(lambda: F.checkpoint_store(x.detach()), "not on a CUDA device")


def test_training_asks_for_the_final_state_only_where_the_caller_does(monkeypatch):
    """It costs a pass over keys and values of its own."""
    from lama_b200 import operators as F
    asked = []

    class Native:
        @staticmethod
        def attention(q, k, v, log_decay, scale, initial_state, lengths, return_state):
            asked.append(return_state)
            return q * 2, q.new_zeros(1, 2, 8, 8) if return_state else None

        @staticmethod
        def attention_backward(grad_o, q, k, v, log_decay, scale, initial_state, lengths, grad_state):
            asked.append(grad_state)
            return grad_o * 2, torch.zeros_like(k), torch.zeros_like(v), None
    monkeypatch.setattr(F, "_native", Native)
    z, ld = torch.ones(1, 4, 2, 8), torch.zeros(2)
    q = z.clone().requires_grad_()
    o = F.linear_attention(q, z, z, ld)
    o.sum().backward()
    assert asked == [False, None] and torch.equal(q.grad, 2 * z)
    q.grad = None
    o, state = F.linear_attention(q, z, z, ld, return_state=True)
    (o.sum() + state.sum()).backward()
    assert asked[2] is True and torch.equal(asked[3], torch.ones_like(state)) and torch.equal(q.grad, 2 * z)


# ------------------------------------------------------------------ pointers at the C ABI

def test_unaligned_pointers_are_refused():
    """A kernel that met one would fault: every pointer is aligned to its elements, workspaces to 16 bytes."""
    from test_operators import attention, call, norm, rows
    p, odd = 4096, 4097

    def check(name, *args, msg="not aligned"):
        rc, text = call(name, *args, 0, None)
        assert rc == EINVAL and msg in text, (name, args, text)
    for kw in (dict(decay=odd), dict(init=odd), dict(lengths=odd)):
        check("lama_linear_attention", attention(**kw), rows(), None, p, 1 << 40)
        check("lama_linear_attention_backward", attention(**kw), rows() * 4 + struct.pack("@2P", 0, 0), p, 1 << 40)
    a = attention(tokens=4096)
    check("lama_linear_attention", a, rows(), odd, p, 1 << 40)
    for w in (4104, odd):
        check("lama_linear_attention", a, rows(), None, w, 1 << 40, msg="workspace is not aligned to 16")
        check("lama_linear_attention_backward", a, rows() * 4 + struct.pack("@2P", 0, 0), w, 1 << 40,
              msg="workspace is not aligned to 16")
    for gs in ((odd, 0), (0, odd)):
        check("lama_linear_attention_backward", a, rows() * 4 + struct.pack("@2P", *gs), p, 1 << 40)
    one = attention(tokens=1)
    check("lama_linear_attention_step", attention(tokens=1, decay=odd), rows(), p, p, 4, None)
    for args in ((odd, odd, 4, None), (p, odd, 4, None), (p, p, 4, odd)):
        check("lama_linear_attention_step", one, rows(), *args)

    none = (None,) * 6
    for kw in (dict(gate=odd), dict(post=odd), dict(pre=odd), dict(scales=odd)):
        check("lama_gated_residual_norm", norm(**kw), p, 64, p, 64, p, p, *none)
    for i in range(4):
        t = [odd if j == i else p for j in range(4)]
        check("lama_gated_residual_norm", norm(), t[0], 64, t[1], 64, t[2], t[3], *none)
    for i in (0, 1, 3, 5):  # post_rstd, pre_rstd and the scales; codes are bytes
        check("lama_gated_residual_norm", norm(), p, 64, p, 64, p, p, *(odd if j == i else p for j in range(6)))
    need, _ = call("lama_gated_residual_norm_workspace", norm())
    fields = ["gu", "gn", "y", "u", "yc", "uc", "ys", "us", "ry", "ru", "gx", "gy", "gg", "gpost", "gpre", "gs"]

    def grads(bad=None):
        v = [odd if f == bad else p for f in fields]
        return struct.pack("@4P4q12P", *v[:4], *(64,) * 4, *v[4:])
    for f in fields:
        if f not in ("yc", "uc"):
            check("lama_gated_residual_norm_backward", norm(), grads(f), p, need)
    check("lama_gated_residual_norm_backward", norm(), grads(), 4104, need, msg="workspace is not aligned to 16")


def test_a_step_refuses_states_that_overlap_in_part():
    """New states over old ones that other threads have yet to read: only the same buffer, or one apart, will do."""
    from test_operators import attention, call, rows
    p, size = 1 << 20, 4 * 2 * 64 * 64 * 4
    for out in (p + 4, p - 4, p + size - 4, p - size + 4):
        rc, text = call("lama_linear_attention_step", attention(tokens=1), rows(), p, out, 4, None, 0, None)
        assert rc == EINVAL and "overlaps" in text, out


# ------------------------------------------------------------------ the device of a report

def test_check_operators_reads_the_current_device(monkeypatch):
    """A device without an index is the current one, as everywhere in torch."""
    from lama_b200 import operators as F
    asked = []

    class Lib:
        def lama_operator_status(self, dev, err, n):
            asked.append(dev)
            return 0
    monkeypatch.setattr(F, "lib", Lib)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 3)
    for d in (None, "cuda", torch.device("cuda"), "cuda:1", 2, torch.device("cuda", 0)):
        F.check_operators(d)
    assert asked == [3, 3, 3, 1, 2, 0]
    refused(lambda: F.check_operators("cpu"), "not a CUDA device")


# ------------------------------------------------------------------ the build

def test_the_library_builds_without_torch(tmp_path):
    """The library and the CLI need no torch: the default target leaves the binding out where there is none, `binding` says so."""
    import os
    import subprocess
    import sys
    csrc = os.path.join(os.path.dirname(__file__), "..", "lama-inpaint-rs_b200", "csrc")

    def make(python, *args):
        return subprocess.run(["make", "-n", "-B", "-C", csrc, f"PYTHON={python}", *args], capture_output=True, text=True)
    bare = tmp_path / "python"
    bare.write_text(f'#!/bin/sh\nexec {sys.executable} -I -S "$@"\n')  # no site-packages: no torch
    bare.chmod(0o755)
    for python in (bare, tmp_path / "missing"):
        r = make(python)
        assert r.returncode == 0 and "liblama_b200.so" in r.stdout and "torch_binding.cpp" not in r.stdout
        assert "not built" in r.stdout
    r = subprocess.run(["make", "-C", csrc, f"PYTHON={bare}", "BINDING=" + str(tmp_path / "b.so"), "binding"],
                       capture_output=True, text=True)
    assert r.returncode != 0 and "needs torch" in r.stdout
    r = make(sys.executable)
    assert r.returncode == 0 and "torch_binding.cpp" in r.stdout
