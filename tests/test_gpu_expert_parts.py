"""A layer of experts split over processes, with a shared expert: one of them has it."""
from __future__ import annotations

import pytest
import torch

from test_gpu_expert_layer import GATE, experts_of, plain_experts

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("has_it", [0, 1, 2])
def test_the_shared_expert_counts_once(dev, has_it):
    from my_int4.decoder import ExpertLayer
    g = torch.Generator().manual_seed(11)
    layer, w = experts_of(g, 16, 4, 256, 128, dev)
    x = torch.randn(70, 256, generator=g).bfloat16().to(dev)
    total = torch.zeros(70, 256, dtype=torch.float64, device=dev)
    for i, (at, n) in enumerate([(0, 4), (4, 6), (10, 6)]):
        part = ExpertLayer(**{**layer.__dict__, "first": at, "up": tuple(t[at:at + n].contiguous() for t in layer.up),
                              "down": tuple(t[at:at + n].contiguous() for t in layer.down),
                              "shared": layer.shared if i == has_it else None})
        total += part(x).double()
    ref = plain_experts(x, w, layer)
    assert float((total.cpu() - ref).norm() / ref.norm()) < GATE
    # the parts and the whole are rounded to bf16 (UNIT 2^-8 of each value), the shared expert's and the routed ones' sums before their own
    whole = layer(x).double()
    assert float((total - whole).norm() / whole.norm()) < 4 * 2.0 ** -8


def test_the_router_sees_all_experts(dev):
    """A process that holds none of a token's choices adds nothing for it."""
    from my_int4.decoder import ExpertLayer
    g = torch.Generator().manual_seed(12)
    layer, w = experts_of(g, 16, 4, 256, 128, dev, shared=False)
    x = torch.randn(40, 256, generator=g).bfloat16().to(dev)
    part = ExpertLayer(**{**layer.__dict__, "first": 12, "up": tuple(t[12:].contiguous() for t in layer.up),
                          "down": tuple(t[12:].contiguous() for t in layer.down)})
    ref = plain_experts(x, w, layer, False, range(12, 16))
    y = part(x).double().cpu()
    none = ref.abs().amax(1) == 0
    assert bool(none.any()) and not bool(y[none].any())
    assert float((y - ref).norm() / ref.norm()) < GATE
