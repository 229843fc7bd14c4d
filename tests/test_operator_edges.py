"""What the token-mixer operators refuse or pass on before any GPU is involved: autograd's demands on the
Python side, pointers and sizes at the C ABI."""

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
