"""Expert layers and rotary heads on the GPU: calls and values at the limits of what they are for.  The bounds are derived beside the plain forms
(tests/_experts.py) and here."""

import pytest
import torch
from torch.autograd import forward_ad

import dynamis_b200 as D
from tests import _experts as X

pytestmark = pytest.mark.gpu


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(gen, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=gen, device="cuda").to(dtype)


def _routing(rows, experts, choices, absent=0.0, seed=1):
    return D.Routing(*X.routing_by_hand(rows, experts, choices, absent, seed, "cuda"))


# ------------------------------------------------------------------------------------------------ forward-mode derivatives
def test_forward_mode_derivatives_are_refused(cuda):
    """There is no formula for them: a tangent raises, also without gradients, and a level that is open changes nothing else."""
    gen = _gen(1)
    q, k, pos, wave = _normal(gen, 20, 2, 8), _normal(gen, 20, 2, 8), _normal(gen, 20, 3), _normal(gen, 4, 3)
    qw, kw = _normal(gen, 8), _normal(gen, 8)
    logits, balance = _normal(gen, 20, 5), _normal(gen, 5)
    routing = _routing(20, 5, 2)
    x, w, b = _normal(gen, 20, 8), _normal(gen, 5, 8, 8), _normal(gen, 5, 8)
    z, r = _normal(gen, 20, 2, 8), _normal(gen, 20, 8)
    by_weights = lambda z, weights, r: D.expert_combine(z, D.Routing(routing.experts, weights, routing.order, routing.start), r)  # noqa: E731
    calls = [(lambda *t: D.rotary_heads(*t)[0], (q, k, pos, wave, qw, kw)), (lambda t, c: D.route_experts(t, 2, bias=c).weights, (logits, balance)),
             (lambda x, w, b: D.expert_linear(x, w, routing, b, "silu"), (x, w, b)), (by_weights, (z, routing.weights, r))]
    for call, args in calls:
        want = call(*args)
        with forward_ad.dual_level():
            assert torch.equal(call(*args), want)
            for i, t in enumerate(args):
                for grad in (True, False):
                    with torch.set_grad_enabled(grad), pytest.raises(RuntimeError, match="jvp"):
                        call(*args[:i], forward_ad.make_dual(t, torch.ones_like(t)), *args[i + 1:])
            assert torch.equal(call(*args), want)
