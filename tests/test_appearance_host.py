"""CPU: the learned-appearance operators' argument checks (before any device
work), and their 64-bit oracle against differences and published vectors."""
import ctypes

import numpy as np
import pytest
import torch

from oracle import appearance as orc
from tidegs_b200 import _lib
from tidegs_b200 import appearance as ap


def _ffn(d=4, h=8, o=3, dtype=torch.float32):
    return (torch.zeros(h, d, dtype=dtype), torch.zeros(h, d, dtype=dtype),
            torch.zeros(o, h, dtype=dtype))


def test_layer_norm_refusals():
    x = torch.zeros(5, 8)
    with pytest.raises(ValueError, match="last dimension"):
        ap.layer_norm(torch.zeros(5, 0))
    with pytest.raises(ValueError, match="last dimension"):
        ap.layer_norm(torch.zeros(2, 8193))
    with pytest.raises(ValueError, match="float64"):
        ap.layer_norm(x.double())
    with pytest.raises(ValueError, match="weight"):
        ap.layer_norm(x, torch.ones(7))
    with pytest.raises(ValueError, match="bias"):
        ap.layer_norm(x, torch.ones(8), torch.zeros(8, dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="bias torch"):
        ap.layer_norm(x.bfloat16(), torch.ones(8), torch.zeros(8, dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="eps"):
        ap.layer_norm(x, eps=-1.0)
    with pytest.raises(RuntimeError, match="no CPU path"):
        ap.layer_norm(x)


def test_gated_feed_forward_refusals():
    x = torch.zeros(5, 4)
    g, u, dn = _ffn()
    with pytest.raises(ValueError, match=r"\[H, D\]"):
        ap.gated_feed_forward(x, g, u[:4], dn)
    with pytest.raises(ValueError, match=r"\[H, D\]"):
        ap.gated_feed_forward(x, g, u, dn.T)
    with pytest.raises(ValueError, match="is not"):
        ap.gated_feed_forward(torch.zeros(5, 3), g, u, dn)
    with pytest.raises(ValueError, match="widths"):
        ap.gated_feed_forward(torch.zeros(5, 257), *_ffn(d=257))
    with pytest.raises(ValueError, match="widths"):
        ap.gated_feed_forward(x, *_ffn(o=300))
    with pytest.raises(ValueError, match="widths"):
        ap.gated_feed_forward(x, *_ffn(h=4097))
    with pytest.raises(ValueError, match="float16"):
        ap.gated_feed_forward(x.half(), *_ffn(dtype=torch.float16))
    with pytest.raises(RuntimeError, match="no CPU path"):
        ap.gated_feed_forward(x, g, u, dn)


def test_dropout_refusals():
    x = torch.zeros(5, 4)
    with pytest.raises(ValueError, match="p 1.5"):
        ap.dropout(x, 1.5, 0)
    with pytest.raises(ValueError, match="p nan"):
        ap.dropout(x, float("nan"), 0)
    with pytest.raises(ValueError, match="seed"):
        ap.dropout(x, 0.5, -1)
    with pytest.raises(ValueError, match="seed"):
        ap.dropout(x, 0.5, 2 ** 64)
    with pytest.raises(ValueError, match="offset"):
        ap.dropout(x, 0.5, 0, offset=2 ** 32)
    with pytest.raises(ValueError, match="offset"):
        ap.dropout(x, 0.5, 0, offset=torch.zeros(2, dtype=torch.int64))
    with pytest.raises(ValueError, match="ids"):
        ap.dropout(x, 0.5, 0, ids=torch.zeros(4, dtype=torch.int64))
    with pytest.raises(ValueError, match="ids"):
        ap.dropout(x, 0.5, 0, ids=torch.zeros(5, dtype=torch.int32))
    with pytest.raises(ValueError, match="values"):
        ap.dropout(torch.zeros(2, 65537), 0.5, 0)
    with pytest.raises(ValueError, match="dimension"):
        ap.dropout(torch.zeros(()), 0.5, 0)
    with pytest.raises(ValueError, match="float64"):
        ap.dropout(x.double(), 0.5, 0)
    with pytest.raises(RuntimeError, match="no CPU path"):
        ap.dropout(x, 0.5, 0)


def test_dropout_refuses_numbers_that_are_not_whole():
    x = torch.zeros(5, 4)
    with pytest.raises(TypeError):
        ap.dropout(x, 0.5, 1.5)
    with pytest.raises(TypeError):
        ap.dropout(x, 0.5, 1, offset=2.5)


def test_unaligned_bfloat16_rows_are_refused_below_python():
    lib = _lib.load()
    f = _lib.FfnArgs()
    f.n, f.d, f.h, f.o, f.dtype = 4, 16, 8, 8, _lib.BF16
    f.x = f.w_gate = f.w_up = f.w_down = f.y = f.scratch = 256
    f.x_stride = 17
    assert lib.tgs_ffn_fwd(ctypes.byref(f), None) == 1 and "aligned" in _lib.last_error()
    f.x_stride, f.x = 16, 258
    assert lib.tgs_ffn_fwd(ctypes.byref(f), None) == 1 and "aligned" in _lib.last_error()
    f.x, f.y = 256, 260
    assert lib.tgs_ffn_fwd(ctypes.byref(f), None) == 1 and "aligned" in _lib.last_error()
    b = _lib.FfnBwdArgs()
    f.y = 256
    b.fwd, b.v_y, b.v_y_stride, b.v_x = f, 256, 12, 256
    assert lib.tgs_ffn_bwd(ctypes.byref(b), None) == 1 and "aligned" in _lib.last_error()
    assert lib.tgs_align_rows(None, 5, 0, 5, None, None) == 0
    assert lib.tgs_align_rows(None, 5, 3, 5, None, None) == 1 and "NULL" in _lib.last_error()
    assert lib.tgs_align_rows(256, 4, 3, 5, 256, None) == 1 and "overlap" in _lib.last_error()


def test_appearance_colors_refusals():
    w = _ffn()
    with pytest.raises(ValueError, match="base"):
        ap.appearance_colors(torch.zeros(5, 3), torch.zeros(4, 4), (None, None), w)
    with pytest.raises(ValueError, match="w_down"):
        ap.appearance_colors(torch.zeros(5, 4), torch.zeros(5, 4), (None, None), w)


def test_entry_points_check_their_arguments():
    lib = _lib.load()
    for name in ("tgs_layer_norm_fwd", "tgs_layer_norm_bwd", "tgs_ffn_fwd", "tgs_ffn_bwd",
                 "tgs_dropout"):
        assert getattr(lib, name)(None, None) == 1
        assert name in _lib.last_error()
    a = _lib.LayerNormArgs()
    a.n, a.c, a.x_stride = 0, 8, 8
    assert lib.tgs_layer_norm_fwd(ctypes.byref(a), None) == 0  # no rows: nothing to do
    a.n = 4
    assert lib.tgs_layer_norm_fwd(ctypes.byref(a), None) == 1 and "NULL" in _lib.last_error()
    a.x, a.x_stride = 256, 7
    assert lib.tgs_layer_norm_fwd(ctypes.byref(a), None) == 1 and "overlap" in _lib.last_error()
    a.c = 8193
    assert lib.tgs_layer_norm_fwd(ctypes.byref(a), None) == 1 and "sizes" in _lib.last_error()
    f = _lib.FfnArgs()
    f.n, f.d, f.h, f.o, f.x_stride, f.dtype = 4, 257, 8, 8, 257, _lib.F32
    assert lib.tgs_ffn_fwd(ctypes.byref(f), None) == 1 and "sizes" in _lib.last_error()
    f.d, f.dtype = 8, _lib.F16
    assert lib.tgs_ffn_fwd(ctypes.byref(f), None) == 1 and "type" in _lib.last_error()
    f.dtype = _lib.BF16
    assert lib.tgs_ffn_fwd(ctypes.byref(f), None) == 1 and "NULL" in _lib.last_error()
    b = _lib.FfnBwdArgs()
    f.x = f.w_gate = f.w_up = f.w_down = 256
    b.fwd, b.v_w_up = f, 256
    assert lib.tgs_ffn_bwd(ctypes.byref(b), None) == 1 and "all given" in _lib.last_error()
    d = _lib.DropoutArgs()
    d.n, d.c, d.x_stride, d.p = 4, 8, 8, 2.0
    assert lib.tgs_dropout(ctypes.byref(d), None) == 1 and "[0, 1]" in _lib.last_error()


def test_struct_offsets_of_the_appearance_arguments(tmp_path):
    import shutil
    import subprocess
    from pathlib import Path

    if shutil.which("gcc") is None:
        pytest.skip("gcc not available")
    lines = ["#include <stdio.h>", "#include <stddef.h>", '#include "tidegs_b200.h"',
             "int main(void) {"]
    expect = []
    for name in ("LayerNormArgs", "LayerNormBwdArgs", "FfnArgs", "FfnBwdArgs", "DropoutArgs"):
        cls = getattr(_lib, name)
        lines.append(f'  printf("%zu\\n", sizeof(Tgs{name}));')
        expect.append(ctypes.sizeof(cls))
        for field, _ in cls._fields_:
            lines.append(f'  printf("%zu\\n", offsetof(Tgs{name}, {field}));')
            expect.append(getattr(cls, field).offset)
    src = tmp_path / "offsets.c"
    src.write_text("\n".join(lines + ["  return 0;", "}"]))
    include = Path(__file__).resolve().parents[1] / "include"
    exe = tmp_path / "offsets"
    subprocess.run(["gcc", "-std=c11", f"-I{include}", str(src), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout
    assert [int(v) for v in out.split()] == expect


# --- the oracle ----------------------------------------------------------------

def test_oracle_gradients_match_differences():
    g = torch.Generator().manual_seed(3)

    def rand(*shape):
        return torch.randn(*shape, generator=g, dtype=torch.float64).requires_grad_(True)

    x, w, b = rand(4, 6), rand(6), rand(6)
    assert torch.autograd.gradcheck(lambda *a: orc.layer_norm(*a), (x, w, b))
    ffn = (rand(4, 5), rand(7, 5), rand(7, 5), rand(3, 7))
    assert torch.autograd.gradcheck(orc.gated_feed_forward, ffn)
    # the closed formulas are autograd's, up to 64-bit rounding
    v = rand(4, 6).detach()
    got = orc.layer_norm_grads(x.detach(), w.detach(), 1e-5, v)
    for a, e in zip(got, torch.autograd.grad(orc.layer_norm(x, w, b), (x, w, b), v)):
        assert torch.allclose(a, e, rtol=1e-12, atol=1e-13)
    v = rand(4, 3).detach()
    got = orc.gated_feed_forward_grads(*(t.detach() for t in ffn), v)
    for a, e in zip(got, torch.autograd.grad(orc.gated_feed_forward(*ffn), ffn, v)):
        assert torch.allclose(a, e, rtol=1e-12, atol=1e-13)


def test_oracle_generator_gives_the_published_words():
    """The known-answer vectors published with Philox4x32-10 (Random123)."""
    ones = 0xFFFFFFFF
    for counter, key, words in (
            ((0, 0, 0, 0), (0, 0), (0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8)),
            ((ones,) * 4, (ones, ones), (0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD)),
            ((0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344), (0xA4093822, 0x299F31D0),
             (0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1))):
        got = orc.philox4x32_10([np.array([c], dtype=np.uint64) for c in counter], key)
        assert tuple(int(w[0]) for w in got) == words


def test_oracle_dropout_depends_on_id_column_and_offset_alone():
    ids = np.array([7, 2 ** 40 + 3, 7, 0])
    keep = orc.dropout_keep(4, 9, 0.5, 11, 5, ids)
    assert np.array_equal(keep[0], keep[2])
    assert np.array_equal(keep[1:2], orc.dropout_keep(1, 9, 0.5, 11, 5, ids[1:2]))
    assert np.array_equal(keep[:, :4], orc.dropout_keep(4, 4, 0.5, 11, 5, ids))
    row = orc.dropout_keep(4, 9, 0.5, 11, 5, ids, per_row=True)
    assert np.array_equal(row, np.repeat(keep[:, :1], 9, 1))
    assert not orc.dropout_keep(4, 9, 1.0, 11).any() and orc.dropout_keep(4, 9, 0.0, 11).all()
