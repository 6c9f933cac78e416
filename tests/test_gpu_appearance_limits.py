"""GPU: the learned-appearance operators at the edges of what their
documentation allows: layouts whose parts start off 16-byte boundaries, widths
at a limit, several host threads, derivatives that are not offered, values near
the ends of their range, sums over very many rows. Tolerances are those of
test_gpu_appearance.py unless a test derives its own."""
import pytest
import torch

from test_gpu_appearance import _ffn_check, _ffn_inputs

pytestmark = pytest.mark.gpu


# --- layouts off 16-byte boundaries ----------------------------------------------

@pytest.mark.parametrize("n,d,h,o", [(5000, 64, 130, 3), (5000, 128, 129, 3), (100, 65, 97, 48), (700, 36, 333, 21),
                                     (9000, 32, 131, 64)])
def test_float32_gradients_whose_slices_are_not_whole_vectors(n, d, h, o):
    """H (2 D + O), or 2 H D, is no multiple of 4 while D or O is one: rows of a
    slice of the weights' gradients start on 16-byte boundaries in some slices
    and off them in others."""
    _ffn_check(*_ffn_inputs(n, d, h, o, torch.float32))
