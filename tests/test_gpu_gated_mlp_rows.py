"""The gated block's forward pass at the edges between its kernels: rows and
columns just within and past what the few-row kernel takes, in both of its
widths, one and several rounds over the input."""
import pytest

torch = pytest.importorskip("torch")

from test_gpu_gated_mlp import TYPES, check_backward, check_forward  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,width,hidden", [(1, 511, 4095), (1, 513, 4097), (8, 512, 4096), (9, 30, 4097), (16, 1025, 4100),
                                               (7, 600, 8191), (8, 33, 8193), (40, 700, 1400), (41, 64, 1430), (128, 520, 17),
                                               (127, 1, 513), (129, 40, 17), (64, 200, 2049), (3, 40, 16390), (17, 64, 8200)])
@pytest.mark.parametrize("ty", TYPES)
@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_forward(gpu, rows, width, hidden, ty, act):
    check_forward(rows, width, hidden, ty, act)


@pytest.mark.parametrize("rows,width,hidden", [(1, 64, 16416), (3, 40, 16390), (31, 64, 16416), (33, 64, 16416)])
@pytest.mark.parametrize("ty", TYPES)
def test_backward_of_few_rows_of_a_wide_block(gpu, rows, width, hidden, ty):
    check_backward(rows, width, hidden, ty, "silu")
