"""The routed experts: which form a call takes, and what fp16 holds of small gradients."""

import pytest
import torch

pytestmark = pytest.mark.gpu

if not torch.cuda.is_available():  # pragma: no cover
    pytest.skip("no CUDA device", allow_module_level=True)

from neural_scaling_weather_b200 import ops  # noqa: E402
from neural_scaling_weather_b200.ops import _ext  # noqa: E402
from tests.test_expert_ops_gpu import BF, DEV, HF, U, expert_exact, expert_inputs, rel  # noqa: E402


@pytest.fixture(autouse=True)
def _no_device_error():
    ext = _ext.require()
    yield
    assert ext.read_error_flag(True) == 0


# experts, width, hidden width, rows an expert, rows of a tile: by more than 5 % the fastest of the three where they were
# timed (the table beside expert_tile), on 148 SMs
TILES = [(2, 768, 1024, 512, 64), (2, 768, 1024, 1024, 256), (2, 1024, 4096, 128, 64), (2, 1024, 4096, 512, 256),
         (1, 1024, 2736, 512, 64), (1, 1024, 2736, 1024, 256), (8, 1024, 2736, 8, 32), (8, 1024, 2736, 64, 64),
         (8, 1024, 2736, 96, 256), (8, 2048, 2736, 64, 64), (8, 2048, 2736, 96, 256), (32, 768, 512, 48, 64),
         (32, 768, 512, 96, 256), (64, 512, 680, 48, 64), (64, 512, 680, 64, 256), (64, 1024, 1368, 16, 32),
         (64, 1024, 1368, 64, 256), (128, 256, 344, 64, 256), (256, 512, 128, 64, 256)]


@pytest.mark.parametrize("E,K,H,rows,tile", TILES)
def test_tiles_are_the_fastest_measured(E, K, H, rows, tile):
    if torch.cuda.get_device_properties(0).multi_processor_count != 148:
        pytest.skip("the rule counts SMs")
    assert _ext.require().expert_tile(rows * E, E, H, K) == tile


@pytest.mark.parametrize("M,E,K,H", [(64, 2, 128, 1024), (200, 2, 64, 4096), (700, 64, 64, 72)])
def test_forms_agree_about_the_rule(M, E, K, H):
    """Either side of the rule's borders, against 64 bits (4 u as in test_expert_ops_gpu.py)."""
    for m in (M, 3 * M, 6 * M):
        x, wt, chosen, w, res, _ = expert_inputs(m, 2, E, K, H, K, BF, seed=m)
        assert rel(ops.expert_mlp(x, wt, chosen, *w, residual=res), expert_exact(x, wt, chosen, w, res, "silu")) < 4 * U[BF]
