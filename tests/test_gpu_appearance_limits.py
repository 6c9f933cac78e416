"""GPU: the learned-appearance operators at the edges of what their
documentation allows: layouts whose parts start off 16-byte boundaries, widths
at a limit, several host threads, derivatives that are not offered, values near
the ends of their range, sums over very many rows. Tolerances are those of
test_gpu_appearance.py unless a test derives its own."""
import ctypes
import subprocess
import sys
import threading
from pathlib import Path

import pytest
import torch

from oracle import appearance as orc
from test_gpu_appearance import HALF, TYPES, U, _far, _ffn_check, _ffn_expect, _ffn_inputs, _gen, _norm_inputs, _rand

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


# --- derivatives that are not offered ------------------------------------------------

def test_forward_mode_is_refused():
    """A dual tensor's tangent is not dropped."""
    from torch.autograd import forward_ad

    from tidegs_b200 import appearance as ap

    x, wg, wu, wd, _ = _ffn_inputs(20, 16, 24, 8, torch.float32)
    w, b = torch.ones(16, device="cuda"), torch.zeros(16, device="cuda")
    calls = [(lambda *a: ap.layer_norm(*a), [x, w, b]), (lambda *a: ap.gated_feed_forward(*a), [x, wg, wu, wd]),
             (lambda a: ap.dropout(a, 0.5, 1), [x])]
    with forward_ad.dual_level():
        for f, args in calls:
            f(*args)  # no tangent: as ever
            for k in range(len(args)):
                dual = [forward_ad.make_dual(t, torch.ones_like(t)) if i == k else t for i, t in enumerate(args)]
                with pytest.raises(RuntimeError, match="forward-mode"):
                    f(*dual)
                with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
                    f(*dual)
                with forward_ad._set_fwd_grad_enabled(False):
                    f(*dual)
            leaf = args[0].detach().requires_grad_(True)
            y = f(leaf, *args[1:])
            v = torch.ones_like(y)
            with pytest.raises(RuntimeError, match="forward-mode"):
                torch.autograd.grad(y, leaf, forward_ad.make_dual(v, v.clone()), retain_graph=True)
            torch.autograd.grad(y, leaf, v)


@pytest.mark.parametrize("transform", ["grad", "jvp", "vmap"])
def test_function_transforms_are_refused(transform):
    from tidegs_b200 import appearance as ap

    x, wg, wu, wd, _ = _ffn_inputs(20, 16, 24, 8, torch.float32)
    for f in (ap.layer_norm, lambda a: ap.gated_feed_forward(a, wg, wu, wd), lambda a: ap.dropout(a, 0.5, 1)):
        with pytest.raises(RuntimeError):
            if transform == "grad":
                torch.func.grad(lambda a: f(a).sum())(x)
            elif transform == "jvp":
                torch.func.jvp(f, (x,), (torch.ones_like(x),))
            else:
                torch.func.vmap(f)(x[:, None])


# --- values near the ends of their range ----------------------------------------------

@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n", [4, 20000])
@pytest.mark.parametrize("d,h,o", [(2, 3, 2), (64, 128, 48), (160, 320, 192)])
def test_closed_gates_of_large_values(dtype, n, d, h, o):
    """silu(-1e25) is -0, so the block is 0 times what passes the gate, however
    large that is; the same for the gate's slope and the gradients."""
    from tidegs_b200 import appearance as ap

    x = torch.zeros(n, d, device="cuda", dtype=dtype)
    x[:, 0], x[:, 1] = -1e25, 1e25
    wg, wu = torch.zeros(2, h, d, device="cuda", dtype=dtype)
    wg[:, 0] = wu[:, 1] = 1.0
    wd = torch.ones(o, h, device="cuda", dtype=dtype)
    leaves = [t.requires_grad_(True) for t in (x, wg, wu, wd)]
    y = ap.gated_feed_forward(*leaves)
    assert not y.any() and not torch.isnan(y).any()
    v = torch.full((n, o), 1e20, device="cuda", dtype=dtype)
    for name, t in zip(("v_x", "v_w_gate", "v_w_up", "v_w_down"), torch.autograd.grad(y, leaves, v)):
        assert not torch.isnan(t).any() and not t.any(), name


# --- several host threads -----------------------------------------------------------

@pytest.mark.parametrize("dtype,sizes", [(torch.float32, [(60, 35, 96, 3), (60, 8, 40, 3)]),
                                         (torch.float32, [(60, 35, 96, 40), (60, 8, 40, 40)]),
                                         (torch.bfloat16, [(60, 256, 512, 256), (60, 16, 16, 16)])])
def test_one_kernel_at_two_sizes_of_shared_memory_from_two_threads(dtype, sizes):
    """Launches of one kernel that want different shared memory, from two host
    threads at once: none is refused, each gives what it gives alone."""
    from tidegs_b200 import _lib
    from tidegs_b200 import appearance as ap

    lib, jobs = _lib.load(), []
    for k, size in enumerate(sizes):
        *ins, _ = _ffn_inputs(*size, dtype, k)
        args, scratch = ap._ffn_args(*ins, backward=False)
        y = torch.empty(size[0], size[3], dtype=dtype, device="cuda")
        args.y = y.data_ptr()
        jobs.append((args, torch.cuda.Stream(), y, ap.gated_feed_forward(*ins), ins, scratch))
    torch.cuda.synchronize()
    start, problems = threading.Barrier(len(jobs)), []

    def run(args, stream):
        start.wait(30)
        for _ in range(20000):
            if lib.tgs_ffn_fwd(ctypes.byref(args), stream.cuda_stream):
                problems.append(_lib.last_error())
                return

    threads = [threading.Thread(target=run, args=job[:2]) for job in jobs]
    for t in threads:
        t.start()
    for t in threads:
        t.join(120)
    torch.cuda.synchronize()
    assert not problems, problems
    for _, _, y, want, *_ in jobs:
        assert torch.equal(y, want)


def test_the_rows_gradient_is_the_same_alone():
    """With the weights' gradients, from one kernel, and without them."""
    from tidegs_b200 import appearance as ap

    x, wg, wu, wd, v = _ffn_inputs(20000, 64, 128, 48, torch.bfloat16)
    leaves = [t.requires_grad_(True) for t in (x, wg, wu, wd)]
    full = torch.autograd.grad(ap.gated_feed_forward(*leaves), leaves, v)[0]
    alone = torch.autograd.grad(ap.gated_feed_forward(x, *(t.detach() for t in leaves[1:])), x, v)[0]
    assert torch.equal(full, alone)


# --- sums over very many rows ---------------------------------------------------------

def test_bfloat16_gradients_of_one_sign_over_many_rows():
    """One slice of rows (4096 hidden values of the widest block leave no SM for
    a second), all products of one sign, so that what additions cut off adds up:
    the mean error of the gradient is what they lose: 8192 values of scattered
    sizes, each rounded to bfloat16 either way by at most 2^-8, shift the mean by
    less than 2^-8 / sqrt(8192) = 4.3e-5. A sum grows evenly over at most 1,024
    instructions, each of which may cut off two units of 2^-23 of what the sum
    is by then: 1,024 / 2 x 2 x 2^-23 = 1.2e-4."""
    from tidegs_b200 import appearance as ap

    n, d, h, o = 300_000, 256, 4096, 256
    g = _gen(5)
    x = torch.rand(n, d, generator=g, device="cuda").bfloat16()
    wg, wu = ((torch.rand(h, d, generator=g, device="cuda") / d * 2 ** torch.randn(h, 1, generator=g, device="cuda"))
              .bfloat16() for _ in range(2))
    wd = (torch.rand(o, h, generator=g, device="cuda") / h).bfloat16().requires_grad_(True)
    v = (torch.rand(n, o, generator=g, device="cuda") * 2 ** torch.randn(o, generator=g, device="cuda")).bfloat16()
    got = torch.autograd.grad(ap.gated_feed_forward(x, wg, wu, wd), wd, v)[0].double()
    cols = slice(0, 32)  # 256 x 32 of the gradient
    want = torch.zeros(o, 32, device="cuda", dtype=torch.float64)
    for r in range(0, n, 50_000):
        rows = x[r:r + 50_000].double()
        hid = orc.silu(rows @ wg[cols].double().T) * (rows @ wu[cols].double().T)
        want += v[r:r + 50_000].double().T @ hid
    assert abs(float((got[:, cols] / want - 1).mean())) < 1.2e-4 + 4.3e-5


def test_bfloat16_gradients_of_more_rows_than_a_sweep():
    """dX and the weights' gradients from one kernel, whose blocks each take more
    tiles than their accumulators hold: products of one sign, so that each result
    is off by its own rounding and the hidden values' at most, twice 2^-8 and the
    product of both."""
    from tidegs_b200 import appearance as ap

    n, d, h, o = 5_300_000, 16, 16, 8
    g = _gen(6)
    x = torch.rand(n, d, generator=g, device="cuda").bfloat16()
    wg, wu, wd = ((torch.rand(*shape, generator=g, device="cuda") / d).bfloat16() for shape in ((h, d), (h, d), (o, h)))
    v = torch.rand(n, o, generator=g, device="cuda").bfloat16()
    leaves = [t.requires_grad_(True) for t in (x, wg, wu, wd)]
    got = torch.autograd.grad(ap.gated_feed_forward(*leaves), leaves, v)
    want = [[], 0, 0, 0]
    deep = [w.detach().double() for w in leaves[1:]]
    for r in range(0, n, 1_000_000):
        v_x, *v_w = orc.gated_feed_forward_grads(x[r:r + 1_000_000].detach().double(), *deep,
                                                 v[r:r + 1_000_000].double())
        want[0].append(v_x)
        want[1:] = [a + b for a, b in zip(want[1:], v_w)]
    want[0] = torch.cat(want[0])
    for a, e in zip(got, want):
        assert float((a.double() / e - 1).abs().max()) <= 2.1 * HALF[torch.bfloat16]


# --- waits that ran out -----------------------------------------------------------------

def test_the_next_call_tells_of_a_wait_that_ran_out():
    """The error word lies where the host reads it without waiting: a call on
    the device that follows such a kernel raises, once (the word is set by hand)."""
    from tidegs_b200 import appearance as ap

    *ins, v = _ffn_inputs(10, 16, 16, 16, torch.bfloat16)
    x = ins[0].requires_grad_(True)
    y = ap.gated_feed_forward(*ins)
    word = ap._err_words[x.device]
    assert not word.is_cuda and word.is_pinned()
    word[0] = 4
    with pytest.raises(RuntimeError, match="timed out"):
        ap.gated_feed_forward(*ins)
    ap.gated_feed_forward(*ins)
    word[0] = 4
    with pytest.raises(RuntimeError, match="timed out"):
        torch.autograd.grad(y, x, v, retain_graph=True)
    torch.autograd.grad(y, x, v)
    word[0] = 4
    with pytest.raises(RuntimeError, match="timed out"):
        ap.check()
    ap.check()


def test_kernels_reach_the_error_word():
    """Another kernel that reports by the same function (an id past a bitmap's
    end, which it skips) writes into it."""
    from tidegs_b200 import _lib
    from tidegs_b200 import appearance as ap

    device = torch.device("cuda", torch.cuda.current_device())
    word = ap._err_word(device)
    bits, ids = torch.zeros(2, dtype=torch.int32, device="cuda"), torch.tensor([3, 5, 64, 7], device="cuda")
    _lib.call("tgs_bitmap_set", bits.data_ptr(), 64, ids.data_ptr(), 4, word.data_ptr(),
              torch.cuda.current_stream().cuda_stream)
    with pytest.raises(RuntimeError, match="index 2"):
        ap.check()
    assert not word.any() and bits.tolist() == [8 + 32 + 128, 0]


def test_a_first_call_under_capture_has_its_error_word():
    _child("""
import torch
from tidegs_b200 import appearance as ap
x, w = torch.randn(300, 32, device="cuda").bfloat16(), torch.randn(32, 32, device="cuda").bfloat16()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    y = ap.gated_feed_forward(x, w, w, w)
word = ap._err_words[x.device]
graph.replay()
ap.check()
assert torch.equal(y, ap.gated_feed_forward(x, w, w, w))
word[0] = 4
try:
    ap.check()
except RuntimeError as e:
    assert "timed out" in str(e)
else:
    raise AssertionError("not told")
""")


def test_first_calls_from_several_threads_share_one_error_word():
    _child("""
import threading, torch
from tidegs_b200 import appearance as ap
device = torch.device("cuda", 0)
torch.zeros(1, device=device)
gate, got = threading.Barrier(8), []
def run():
    gate.wait()
    got.append(ap._err_word(device).data_ptr())
threads = [threading.Thread(target=run) for _ in range(8)]
[t.start() for t in threads]
[t.join() for t in threads]
assert len(got) == 8 and len(set(got)) == 1 and got[0] == ap._err_words[device].data_ptr(), got
""")


# --- a row's result is its own --------------------------------------------------------

@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("d,h,o", [(32, 64, 3), (64, 128, 48), (128, 384, 128), (200, 40, 30), (256, 512, 256)])
def test_a_row_gives_the_same_bits_in_calls_of_any_size(dtype, d, h, o):
    """A Gaussian's color does not depend on how many others the call holds; its
    gradient, in bfloat16, only on whether they are more than 18,944."""
    from tidegs_b200 import appearance as ap

    x, wg, wu, wd, v = _ffn_inputs(40000, d, h, o, dtype)
    ws = [w.requires_grad_(True) for w in (wg, wu, wd)]

    def run(k, weights):
        rows = x[:k].detach().requires_grad_(True)
        y = ap.gated_feed_forward(rows, *weights)
        return y.detach(), torch.autograd.grad(y, [rows, *(w for w in weights if w.requires_grad)], v[:k])[0]

    whole, most = run(40000, ws), run(18944, ws)
    for k in (1, 200, 18944, 18945, 30001):
        for weights in (ws, [w.detach() for w in ws]):
            y, v_x = run(k, weights)
            assert torch.equal(y, whole[0][:k])
            assert torch.equal(v_x, (whole if k > 18944 or dtype == torch.float32 else most)[1][:k])


@pytest.mark.parametrize("n,d,h,o", [(18945, 35, 96, 3), (20011, 64, 128, 48), (50000, 145, 72, 9),
                                     (30000, 256, 512, 256)])
def test_large_bfloat16_calls_round_their_outputs_once(n, d, h, o):
    from tidegs_b200 import appearance as ap

    *ins, v = _ffn_inputs(n, d, h, o, torch.bfloat16, 3)
    _far(ap.gated_feed_forward(*ins), _ffn_expect(*ins, v, torch.bfloat16, parts=2)["y"], "y")


# --- every row counts -------------------------------------------------------------

@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,d,h,o", [(60000, 256, 192, 256), (50000, 130, 129, 200), (60000, 64, 40, 64),
                                     (40003, 64, 128, 48)])
def test_every_tile_of_rows_enters_the_weight_gradients(dtype, n, d, h, o):
    """Row r's inputs are zero but in column (r / 128) % D, its gradients but in
    column (r / 128) % O: a column of the weights' gradients sums few rows, and
    its bound is those rows', so that a lost or doubled tile is seen."""
    from tidegs_b200 import appearance as ap

    x, wg, wu, wd, v = _ffn_inputs(n, d, h, o, dtype)
    tile = torch.arange(n, device="cuda") // 128
    x = x.abs() + 0.5
    v = v.abs() + 0.05
    x = torch.where((tile % d)[:, None] == torch.arange(d, device="cuda"), x, 0).to(dtype)
    v = torch.where((tile % o)[:, None] == torch.arange(o, device="cuda"), v, 0).to(dtype)
    leaves = [t.requires_grad_(True) for t in (x, wg, wu, wd)]
    _, got_g, got_u, got_d = torch.autograd.grad(ap.gated_feed_forward(*leaves), leaves, v)
    args = [t.detach() for t in leaves]
    for k in range(max(d, o)):
        if k < d:
            rows = (tile % d == k).nonzero()[:, 0]
            want = _ffn_expect(args[0][rows], *args[1:], v[rows], dtype)
            _far(got_g[:, k], _column(want["v_w_gate"], k), f"v_w_gate, column {k}")
            _far(got_u[:, k], _column(want["v_w_up"], k), f"v_w_up, column {k}")
        if k < o:
            rows = (tile % o == k).nonzero()[:, 0]
            want = _ffn_expect(args[0][rows], *args[1:], v[rows], dtype)["v_w_down"]
            _far(got_d[k], _column(want.T, k), f"v_w_down, row {k}")


def _column(want, k):
    return type(want)(want.val[:, k], want.err[:, k])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,c", [(50001, 768), (50001, 59), (30000, 64), (20000, 1025)])
def test_every_row_enters_the_norm_gradients(dtype, n, c):
    """Row r's gradient is zero but in column (r / 8) % C."""
    from tidegs_b200 import appearance as ap

    x, w, b, v = _norm_inputs(n, c, dtype, torch.float32)
    on = (torch.arange(n, device="cuda") // 8 % c)[:, None] == torch.arange(c, device="cuda")
    v = torch.where(on, v.abs() + 0.05, 0).to(dtype)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    _, got_w, got_b = torch.autograd.grad(ap.layer_norm(*leaves), leaves, v)
    # the sums' bounds by the rows that count: zeros add exactly
    most = int(on.sum(0).max())
    x64, v64 = x.detach().double(), v.double()
    dev = x64 - x64.mean(1, keepdim=True)
    std = torch.sqrt((dev * dev).mean(1, keepdim=True) + 1e-5)
    z = dev / std
    unit = (c + 16) * U * (1 + x64.abs().amax(1, keepdim=True) / std)
    want_w, want_b = (v64 * z).sum(0), v64.sum(0)
    z_err = unit * (1 + z.abs())
    err_w = (v64 * z_err).sum(0) + (most + 4) * U * (v64 * (z.abs() + z_err)).sum(0)
    assert bool(((got_w.double() - want_w).abs() <= err_w + HALF[torch.float32] * want_w.abs()).all())
    assert bool(((got_b.double() - want_b).abs() <= (most + 4) * U * want_b).all())


@pytest.mark.parametrize("n,d,h,o", [(3000, 256, 512, 256), (60000, 128, 256, 128), (5000, 35, 96, 3)])
def test_float32_errors_as_a_whole(n, d, h, o):
    """The 2-norm of the error. A result's sums run through H (or D, or n)
    terms; on the fp32 pipes each addition is off by at most 2^-24 of the
    partial sum, at random: sqrt(K) 2^-24 / sqrt(3) of the terms' spread, as
    large as the result's: 4e-7 at 512. On the tensor cores a piece of 64 loses up
    to 8 x 2^-24 in the additions of its largest products and 2^-24 more in those
    of the smaller ones, 5.4e-7 at most. Three such products follow one another,
    each with its own errors: sqrt(3) x 5.4e-7 = 9.3e-7."""
    from tidegs_b200 import appearance as ap

    *ins, v = _ffn_inputs(n, d, h, o, torch.float32)
    leaves = [t.requires_grad_(True) for t in ins]
    y = ap.gated_feed_forward(*leaves)
    got = (y.detach(), *torch.autograd.grad(y, leaves, v))
    deep = [t.detach().double() for t in ins]
    want = (orc.gated_feed_forward(*deep), *orc.gated_feed_forward_grads(*deep, v.double()))
    for a, e in zip(got, want):
        assert float((a.double() - e).norm() / e.norm()) < 1e-6


@pytest.mark.parametrize("dtype", TYPES)
def test_dropout_of_whole_rows_with_strides(dtype):
    from tidegs_b200 import appearance as ap

    wide = _rand(_gen(6), 90, 72, dtype=dtype)
    ids = torch.arange(180, device="cuda")[::2] * 7 + 2 ** 35
    for x in (wide[:, 8:40], wide[:, 1:34], wide[::2, :32], wide[:, ::2], wide[:40].T, wide[:1].expand(90, 72)):
        who = ids[:x.shape[0]]
        got = ap.dropout(x, 0.4, 8, offset=2, ids=who, per_row=True)
        assert torch.equal(got, ap.dropout(x.contiguous(), 0.4, 8, offset=2, ids=who.contiguous(), per_row=True))
        kept = torch.from_numpy(orc.dropout_keep(x.shape[0], 1, 0.4, 8, 2, who.cpu().numpy())).cuda()
        assert torch.equal(got != 0, kept & (x != 0))


# --- accounts -----------------------------------------------------------------------

def test_launches_are_counted():
    """The kernels that a call launched, by the plans of the different forms."""
    from tidegs_b200 import _lib
    from tidegs_b200 import appearance as ap

    def count(f):
        before = _lib.launch_counter["kernels"]
        f()
        return _lib.launch_counter["kernels"] - before

    def ffn(n, d, h, o, dtype, grads):
        *ins, v = _ffn_inputs(n, d, h, o, dtype)
        leaves = [t.requires_grad_(grads in ("all", k)) for k, t in zip(("x", "", "", ""), ins)]
        if not grads:
            with torch.no_grad():
                return count(lambda: ap.gated_feed_forward(*leaves))
        y = ap.gated_feed_forward(*leaves)
        return count(lambda: torch.autograd.grad(y, [t for t in leaves if t.requires_grad], v))

    f32, b16 = torch.float32, torch.bfloat16
    assert ffn(100, 35, 96, 3, f32, "") == 1
    assert ffn(100, 35, 96, 3, f32, "x") == 1
    assert ffn(100, 35, 96, 3, f32, "all") == 3            # dX, weights, their sum
    assert ffn(100, 128, 256, 128, f32, "") == 5           # three splits, hidden values, output
    assert ffn(100, 128, 256, 128, f32, "all") == 8        # four splits, hidden, dX, weights, their sum
    assert ffn(100, 64, 128, 48, b16, "") == 1
    assert ffn(100, 256, 512, 256, b16, "") == 2           # weights laid out before
    assert ffn(100, 256, 512, 256, b16, "all") == 4        # and dX, weights, their sum
    x, w, b, v = _norm_inputs(50, 40, f32, f32)
    x.requires_grad_(True)
    y = ap.layer_norm(x, w, b)
    assert count(lambda: torch.autograd.grad(y, x, v, retain_graph=True)) == 1
    w.requires_grad_(True)
    y = ap.layer_norm(x, w, b)
    assert count(lambda: torch.autograd.grad(y, (x, w), v)) == 2
