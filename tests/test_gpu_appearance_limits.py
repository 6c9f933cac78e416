"""GPU: the learned-appearance operators at the edges of what their
documentation allows: layouts whose parts start off 16-byte boundaries, widths
at a limit, several host threads, derivatives that are not offered, values near
the ends of their range, sums over very many rows. Tolerances are those of
test_gpu_appearance.py unless a test derives its own."""
import subprocess
import sys
from pathlib import Path

import pytest
import torch

from test_gpu_appearance import _ffn_check, _ffn_inputs

pytestmark = pytest.mark.gpu

HERE = Path(__file__).resolve().parent


def _child(code):
    """Runs `code` in a process of its own (nothing of this one's CUDA state)."""
    head = f"import sys; sys.path[:0] = [{str(HERE.parent)!r}, {str(HERE)!r}]\n"
    done = subprocess.run([sys.executable, "-c", head + code], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stdout[-2000:] + done.stderr[-2000:]


# --- layouts off 16-byte boundaries ----------------------------------------------

@pytest.mark.parametrize("n,d,h,o", [(5000, 64, 130, 3), (5000, 128, 129, 3), (100, 65, 97, 48), (700, 36, 333, 21),
                                     (9000, 32, 131, 64)])
def test_float32_gradients_whose_slices_are_not_whole_vectors(n, d, h, o):
    """H (2 D + O), or 2 H D, is no multiple of 4 while D or O is one: rows of a
    slice of the weights' gradients start on 16-byte boundaries in some slices
    and off them in others."""
    _ffn_check(*_ffn_inputs(n, d, h, o, torch.float32))


# --- widths at a limit -------------------------------------------------------------

def test_layer_norm_backward_where_shared_memory_passes_its_default():
    """Two sums a column, 48 KB at 6144 columns, beside the kernel's own few
    bytes; ascending, so that no wider call comes first."""
    _child("""
import torch
from test_gpu_appearance import TYPES, _norm_check, _norm_inputs
for dtype in TYPES:
    for c in (6136, 6140, 6141, 6143, 6144, 6145, 6152):
        _norm_check(*_norm_inputs(3, c, dtype, dtype))
""")
