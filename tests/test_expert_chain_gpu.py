"""The routed experts' launches, captured once and replayed on choices that change from replay to replay: every kernel of
the chain must see what the one before it has just written (the same addresses hold another sorting each time)."""

import pytest
import torch

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():  # pragma: no cover
    pytest.skip("no CUDA device", allow_module_level=True)

from neural_scaling_weather_b200 import ops  # noqa: E402
from neural_scaling_weather_b200.ops import _ext  # noqa: E402

DEV = torch.device("cuda")
BF = torch.bfloat16


# tokens, choices, experts, widths: tiles of 32, 64 and 256 rows behind the sorting in one launch, and in three
@pytest.mark.parametrize("M,k,E,K,H", [(37, 2, 16, 256, 136), (150, 2, 4, 128, 344), (2000, 2, 2, 128, 1024),
                                       (5000, 2, 3, 128, 1024)])
@pytest.mark.parametrize("train", [False, True])
def test_replays_see_their_own_choices(M, k, E, K, H, train):
    g = torch.Generator(device=DEV).manual_seed(M)
    x = torch.randn(M, K, generator=g, device=DEV).to(BF)
    w = [(torch.randn(*s, generator=g, device=DEV) * s[-1] ** -0.5).to(BF).requires_grad_(train)
         for s in ((E, H, K), (E, H, K), (E, K, H))]
    chosen = torch.randint(-1, E, (M, k), generator=g, device=DEV)
    weights = torch.rand(M, k, generator=g, device=DEV, dtype=torch.float32)

    def step():
        if not train:
            return [ops.expert_mlp(x, weights, chosen, *w, residual=x)]
        y = ops.expert_mlp(x, weights, chosen, *w, residual=x)
        return [y.detach(), *torch.autograd.grad(y, w, x)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(12):
        # all to one expert, none at all, and random ones by turns
        chosen.copy_(torch.full_like(chosen, i % E) if i % 4 == 1 else torch.full_like(chosen, -1) if i % 4 == 3
                     else torch.randint(-1, E, (M, k), generator=g, device=DEV))
        x.copy_(torch.randn(M, K, generator=g, device=DEV))
        graph.replay()
        got = [t.clone() for t in out]
        for a, b in zip(got, step()):
            assert torch.equal(a, b), i
        if i % 4 == 3:
            assert torch.equal(got[0], x)
    assert _ext.require().read_error_flag(True) == 0
