"""The e4m3 product: what its kernels wait on, the binding's checks of its epilogue, every output of the kernel on CTA
pairs against 64 bits.  Tolerances are those of test_fp8_block.py."""
import gc
import math
import os
import re
import subprocess
import sys
import threading
import weakref

import pytest
import torch

from conftest import PKG
from test_fp8_block import ACTS, F8, U32, blank, blocked, fp8_operand, linear64, randn, run_linear


# ---------------------------------------------------------------------------------------------------- waits have an end
def gemm_source():
    with open(os.path.join(PKG, "csrc", "edb200_fp8_gemm.cu")) as fh:
        return re.sub(r"//[^\n]*", "", fh.read())


def test_no_barrier_among_some_of_the_warps():
    """A warp whose wait has given up goes to the end of the kernel.  Others may have seen the same phase complete: a barrier
    among them without a limit would wait for that warp for good.  So between set-up and teardown, where every
    thread arrives, there is none; mbarrier waits have a limit."""
    assert not re.search(r"named_bar_sync|bar\.sync|barrier\.sync|barrier\.cta", gemm_source())


def test_a_warp_gives_up_as_one():
    """A lane that leaves a loop alone leaves the others at elect.sync, or at a load from tensor memory, for good.  So a wait is
    voted on by its warp, or made by one lane in a loop without any instruction for the whole warp."""
    src, rest = gemm_source(), ""
    blocks = []
    while (at := src.find("if (elect_one()) {")) >= 0:
        depth, end = 1, at + len("if (elect_one()) {")
        while depth:
            depth += {"{": 1, "}": -1}.get(src[end], 0)
            end += 1
        blocks.append(src[at + len("if (elect_one()) {"):end])
        rest, src = rest + src[:at], src[end:]
    rest += src
    waits = re.compile(r"\bmbar_wait\(")
    assert sum(len(waits.findall(b)) for b in blocks) >= 6 and "mbar_wait_warp(" in rest
    assert not waits.search(rest)
    for b in blocks:
        assert not re.search(r"__syncwarp|__all_sync|__shfl|__any_sync|elect_one|mbar_wait_warp|tmem_ld|tmem_wait|__syncthreads", b)


def test_nothing_plain_is_shared_between_calls():
    """Entry points may be called from several threads: what a function keeps between calls is atomic."""
    for name in ("fp8_gemm", "fp8_quant", "block_norm", "rope"):
        with open(os.path.join(PKG, "csrc", f"edb200_{name}.cu")) as fh:
            kept = re.findall(r"^[ \t]+static (?!const\b|constexpr\b)([^=;{]*)", fh.read(), re.M)
        assert all("atomic" in k or "PerDevice" in k for k in kept), (name, kept)


# ------------------------------------------------------------------------------------------------ epilogues that do not fit
def product(edb, m=4, k=256, n=130, **ep):
    """A product's arguments on the CPU, as far as the checks go; ep is built over them."""
    z = torch.zeros
    args = dict(w=edb.Fp8Weight(z(n, k, dtype=F8), z(-(-n // 128), 2)), x=z(m, k, dtype=F8), x_scale=z(m, 2))
    return args, edb.make_epilogue(**{**dict(out=z(4, 144)[:, :130]), **ep})


def test_epilogue_refusals(edb):
    z = torch.zeros
    gated = dict(gate=z(130), residual=z(4, 130))
    for ep, text in (
        (dict(out=z(3, 130)), "out must hold 4 rows"), (dict(out=z(4, 128)), "out must hold 4 rows"),
        (dict(out=z(4, 129)), "out must hold"), (dict(out=z(130)), "out must hold"), (dict(out=z(130, 4).t()), "out must hold"),
        (dict(out=z(3, 144), ldo=160), "out must hold"), (dict(bias=z(129)), "bias"), (dict(bias=z(131)), "bias"),
        (dict(bias=z(130, dtype=torch.float16)), "bias"), (dict(bias=z(260)[::2]), "bias"), (dict(gated, gate=z(128)), "gate"),
        (dict(gated, gate=z(130, dtype=torch.bfloat16)), "gate"), (dict(gated, residual=z(3, 130)), "residual must hold"),
        (dict(gated, residual=z(4, 120)), "residual must hold"), (dict(gated, residual=z(4, 130, dtype=torch.float16)), "residual"),
    ):
        args, e = product(edb, **ep)
        with pytest.raises(ValueError, match=text):
            edb.mul_mat_fp8(ep=e, **args)


def test_epilogue_kept_for_longer_rows_is_refused(edb):
    """What was checked for four rows does not pass for five, nor for another weight."""
    _, e = product(edb)
    edb._check_epilogue(e, 4, 130, -1)
    assert e.fits == (4, 130, -1)
    for m, n in ((5, 130), (4, 145)):
        args, _ = product(edb, m=m, n=n)
        with pytest.raises(ValueError, match="out must hold"):
            edb.mul_mat_fp8(ep=e, **args)


def test_epilogues_that_fit(edb):
    """A row alone, fewer rows than the buffer, a stride of the caller's, a residual that no gate asks for, addresses set by hand."""
    z = torch.zeros
    for m, ep in ((1, dict(out=z(130))), (4, dict(out=z(4, 144))), (2, dict(out=z(4, 130))), (4, dict(out=z(4, 2, 65))), (4, dict(out=z(4 * 144), ldo=144)),
                  (4, dict(residual=z(2, 2, dtype=torch.float16))), (4, dict(bias=z(1, 130)))):
        edb._check_epilogue(product(edb, **ep)[1], m, 130, -1)
    by_hand = product(edb, out=z(1, 130))[1]
    by_hand.out = z(9, 144).data_ptr()
    edb._check_epilogue(by_hand, 9, 130, -1)
    raw = edb.Epilogue()
    assert raw.tensors is None and by_hand.tensors is not None


def test_epilogue_keeps_its_tensors(edb):
    bias = torch.zeros(130)
    seen = weakref.ref(bias)
    _, e = product(edb, bias=bias)
    del bias
    gc.collect()
    assert seen() is not None and seen().data_ptr() == e.bias
    del e, _
    gc.collect()
    assert seen() is None


@pytest.mark.gpu
def test_epilogue_places(edb, cuda):
    """Every tensor of the epilogue on the current device; a kept epilogue serves fewer rows and leaves the others."""
    k, n = 256, 130
    xq, xs = fp8_operand(6, k, 1, 1)
    w = edb.Fp8Weight(*fp8_operand(n, k, 128, 2))
    out, res, gate, bias = blank(6, n, torch.float32), randn(6, 144)[:, :n], randn(n), randn(n)
    good = dict(out=out, residual=res, gate=gate, bias=bias)
    for name in good:
        with pytest.raises(ValueError, match=f"{name} is on cpu"):
            edb.mul_mat_fp8(w, xq, xs, edb.make_epilogue(**{**good, name: good[name].cpu()}))
    ep = edb.make_epilogue(**good)
    edb.mul_mat_fp8(w, xq, xs, ep)
    whole = out.clone()
    out.fill_(5.0)
    edb.mul_mat_fp8(w, xq[:2], xs[:2], ep)
    assert torch.equal(out[:2], whole[:2]) and bool((out[2:] == 5.0).all())


# ------------------------------------------------------------------------------------------- every output of the pair kernel
# Ragged in both directions, one to nine blocks of 128 k, n no multiple of 4.  The pairs take what would be several waves of 128 x
# 128 tiles; the shapes of one wave (the first two and the fourth) lie just below.
PAIR_SHAPES = [(600, 72, 3333), (600, 1024, 3330), (2600, 300, 1001), (515, 1100, 3607),
               (1290, 72, 2891), (1290, 1024, 2890), (1283, 1100, 2895), (2600, 300, 4001)]
OUTS = [torch.float32, torch.float16, torch.bfloat16, "gated", "f8"]


@pytest.mark.gpu
@pytest.mark.parametrize("m,k,n", PAIR_SHAPES)
@pytest.mark.parametrize("out", OUTS)
@pytest.mark.parametrize("bias", [True, False])
def test_pair_outputs(edb, cuda, m, k, n, out, bias):
    run_linear(edb, m, k, n, out, bias=bias, pad=16 if m % 2 else 0, seed=m + k)


@pytest.mark.gpu
@pytest.mark.parametrize("act", sorted(ACTS))
@pytest.mark.parametrize("bias", [True, False])
@pytest.mark.parametrize("out", OUTS)
def test_pair_activations(edb, cuda, act, bias, out):
    run_linear(edb, 700, 200, 3402, out, act=act, bias=bias, seed=7)


@pytest.mark.gpu
@pytest.mark.parametrize("m,k,n", PAIR_SHAPES)
def test_pair_residual_in_place(edb, cuda, m, k, n):
    run_linear(edb, m, k, n, "gated", in_place=True, pad=16, seed=k)


@pytest.mark.gpu
@pytest.mark.parametrize("out", ["f8", "gated", torch.bfloat16])
def test_pair_tiles_in_chunks(edb, cuda, out):
    """k so long that 13 of the 21 feature tiles are walked together: a second, narrower chunk."""
    run_linear(edb, 300, 13824, 5200, out, act="gelu_tanh", seed=3)


@pytest.mark.gpu
@pytest.mark.parametrize("out", ["f8", "gated", torch.bfloat16])
def test_pair_tiles_in_chunks_of_many_rows(edb, cuda, out):
    """The same with several token tiles for each of the features'."""
    run_linear(edb, 1300, 13824, 5200, out, act="gelu_tanh", seed=4)


@pytest.mark.gpu
@pytest.mark.parametrize("out", [torch.float16, "f8"])
@pytest.mark.parametrize("m,k,n", [
    (1, 512, 1000), (12, 700, 4300), (40, 1536, 4400), (64, 768, 9000),      # few rows: parts of three blocks and more
    (192, 1536, 768), (129, 1792, 300), (321, 1536, 250),                    # few-row clusters beyond 64 rows
    (129, 5120, 700), (300, 5120, 1500), (128, 5120, 2304), (150, 640, 2300),   # tiles in eight, four and two parts
    (384, 640, 4400), (257, 1280, 10300), (96, 640, 9400), (100, 300, 13000)])  # in one; pairs that would be half empty
def test_where_the_choice_of_kernel_changes(edb, cuda, m, k, n, out):
    run_linear(edb, m, k, n, out, seed=m + n)


@pytest.mark.gpu
@pytest.mark.parametrize("m,k,n", [(3, 200, 77), (90, 200, 130), (700, 200, 3402)])
def test_bias_and_gate_need_no_alignment(edb, cuda, m, k, n):
    xq, xs = fp8_operand(m, k, 1, 1)
    wq, ws = fp8_operand(n, k, 128, 2, 0, 0.05)
    bias, gate, res = randn(n + 1, seed=3), randn(n + 3, seed=4), blank(m, n, torch.float32, fill=2.0)
    y = [blank(m, n, torch.float32) for _ in range(2)]
    w = edb.Fp8Weight(wq, ws)
    edb.mul_mat_fp8(w, xq, xs, edb.make_epilogue(y[0], bias=bias[1:], gate=gate[3:], residual=res))
    edb.mul_mat_fp8(w, xq, xs, edb.make_epilogue(y[1], bias=bias[1:].clone(), gate=gate[3:].clone(), residual=res))
    assert torch.equal(*y)


@pytest.mark.gpu
@pytest.mark.parametrize("out", [torch.float32, "f8"])
def test_pair_is_the_same_every_run_and_row_by_row(edb, cuda, out):
    """The same bits again, and a NaN row or scale stays in its row."""
    m, k, n = 1000, 640, 2570
    xq, xs = fp8_operand(m, k, 1, 3)
    w = edb.Fp8Weight(*fp8_operand(n, k, 128, 4))

    def run():
        y = torch.zeros(m, 2576, device="cuda", dtype=F8 if out == "f8" else out)[:, :n]
        ys = torch.zeros(m, 21, device="cuda") if out == "f8" else None
        edb.mul_mat_fp8(w, xq, xs, edb.make_epilogue(y), ys)
        return (y.float(), ys) if out == "f8" else (y, y[:, :1].clone())

    first, first_scale = run()
    for _ in range(5):
        again, scale = run()
        assert torch.equal(again, first) and torch.equal(scale, first_scale)
    rows = torch.zeros(m, dtype=torch.bool, device="cuda")
    for bad in (0, 127, 128, 500, 999):
        rows[bad] = True
        if bad % 2:
            xs[bad, 1] = float("nan")
        else:
            xq[bad, 5] = float("nan")
    got, scale = run()
    assert bool(torch.isnan(got[rows]).all())
    assert torch.equal(got[~rows], first[~rows]) and torch.equal(scale[~rows], first_scale[~rows])


@pytest.mark.gpu
def test_pair_quantised_output_of_rows_not_finite(edb, cuda):
    """An infinity in a row's activated block reaches the next product as NaN, and its neighbours keep their scale."""
    m, k, n = 1100, 256, 2570
    xq, xs = fp8_operand(m, k, 1, 3)
    wq, ws = fp8_operand(n, k, 128, 4)
    bias = torch.zeros(n, device="cuda")
    bias[3], bias[300], bias[2569] = float("inf"), float("-inf"), float("inf")
    y, ys = blank(m, n, F8), torch.empty(m, 21, device="cuda")
    edb.mul_mat_fp8(edb.Fp8Weight(wq, ws), xq, xs, edb.make_epilogue(y, bias=bias), ys)
    plain, _ = linear64(xq, xs, wq, ws, None, "none")
    lost = torch.isinf(bias)
    assert torch.equal(torch.isnan(y.float()), lost[None].expand(m, n))
    plain[:, lost] = 0.0
    top = blocked(plain, 1, torch.float64).abs().amax((1, 3))
    assert bool(((ys.double() * 448 - top).abs() <= top * 2.0 ** -12).all())


@pytest.mark.gpu
def test_pair_on_two_streams_and_in_two_recordings_at_once(edb, cuda):
    m, k, n = 1000, 1280, 2600
    xq, xs = fp8_operand(m, k, 1, 1)
    w = edb.Fp8Weight(*fp8_operand(n, k, 128, 2, 0, 0.05))
    bias = randn(n, seed=5)
    outs = [torch.empty(m, 2608, device="cuda")[:, :n] for _ in range(5)]
    eps = [edb.make_epilogue(o, bias=bias) for o in outs]
    edb.mul_mat_fp8(w, xq, xs, eps[4])
    torch.cuda.synchronize()
    streams, graphs = [torch.cuda.Stream(), torch.cuda.Stream()], []
    for i, st in enumerate(streams):
        with torch.cuda.stream(st):
            graphs.append(edb.Graph(lambda i=i: edb.mul_mat_fp8(w, xq, xs, eps[i])))
    for _ in range(20):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                graphs[i].launch()
                edb.mul_mat_fp8(w, xq, xs, eps[2 + i])
    torch.cuda.synchronize()
    edb.poll_status()
    for o in outs[:4]:
        assert torch.equal(o, outs[4])


@pytest.mark.gpu
def test_steps_of_a_quantised_output_lie_at_borders(edb, cuda):
    """Context rows through a whole up-projection: a byte is another than 64 bits give only where the value lies within the
    f32 sum's error of the border between the two."""
    run_linear(edb, 154, 1536, 6144, "f8", act="gelu_tanh", seed=11)


# ------------------------------------------------------------------------------------------- activations far from zero
@pytest.mark.gpu
@pytest.mark.parametrize("m", [3, 90, 700, 2900])
@pytest.mark.parametrize("act", ["gelu_erf", "gelu_tanh", "silu"])
def test_activations_of_negative_values_keep_their_relative_error(edb, cuda, m, act):
    """Rows of zeros and a bias: the activation's argument is exact, and its value is compared relative to itself.

    u = 2^-24, and each constant and operation rounds once unless said.  gelu_erf: -v^2 / 2 by three roundings makes
    1.5 v^2 u of the exponential, its approximation 3 u (2^-22.5); t = 1 / (1 + 0.305 |v|) is off by 5 u (the fast division by 2
    steps), which h turns into at most 2.62 times as much; the polynomial's sums 3.1 u, its fit 1.7 u, three products:
    (24 + 1.5 v^2) u.  silu: __expf(x) by 2 + 1.173 |x| steps of 2 u, the sum by u, the fast division by 4 u:
    (9 + 2.35 |v|) u.  gelu_tanh: its exponent t takes six roundings besides: (9 + 8.35 |t|) u."""
    n = 2602
    low, high = {"gelu_erf": (-12.0, 6.0), "gelu_tanh": (-9.0, 9.0), "silu": (-85.0, 20.0)}[act]
    v = torch.linspace(low, high, n, device="cuda")
    w = edb.Fp8Weight(torch.zeros(n, 128, device="cuda", dtype=F8), torch.ones(21, 1, device="cuda"))
    y = blank(m, n, torch.float32)
    edb.mul_mat_fp8(w, torch.zeros(m, 128, device="cuda", dtype=F8), torch.ones(m, 1, device="cuda"),
                    edb.make_epilogue(y, bias=v, act=ACTS[act]))
    x = v.double()
    t = 2 * math.sqrt(2 / math.pi) * (x + 0.044715 * x ** 3)
    want, roundings = {"gelu_erf": (0.5 * x * torch.erfc(-x / math.sqrt(2)), 24 + 1.5 * x * x),
                       "gelu_tanh": (x * torch.sigmoid(t), 9 + 8.35 * t.abs()),
                       "silu": (x * torch.sigmoid(x), 9 + 2.35 * x.abs())}[act]
    off = (y.double() - want).abs() / (want.abs() * U32 * roundings * (1 + 2.0 ** -10))
    assert bool((off[:, want != 0] <= 1).all()), off.nan_to_num().max().item()


# ------------------------------------------------------------------------------------------------------ threads of their own
@pytest.mark.gpu
@pytest.mark.parametrize("m", [8, 300, 2600])
def test_call_from_a_thread_of_its_own(edb, cuda, m):
    """A thread that has made no CUDA call yet has no current context: the tensor maps are made all the same."""
    k, n = 256, 1100
    xq, xs = fp8_operand(m, k, 1, 1)
    w = edb.Fp8Weight(*fp8_operand(n, k, 128, 2))
    y = [torch.zeros(m, 1104, device="cuda")[:, :n] for _ in range(2)]
    edb.mul_mat_fp8(w, xq, xs, edb.make_epilogue(y[0]))
    torch.cuda.synchronize()
    failed = []

    def work():
        try:
            edb.mul_mat_fp8(w, xq, xs, edb.make_epilogue(y[1]))
        except Exception as e:
            failed.append(e)

    t = threading.Thread(target=work)
    t.start()
    t.join()
    torch.cuda.synchronize()
    assert not failed, failed
    assert torch.equal(*y)


FIRST_CALLS = """
import sys, threading
import torch
sys.path.insert(0, sys.argv[1])
import conftest
edb = conftest.load_pkg_module("edb200")
cases = []
for m, n in ((8, 400), (30, 400), (60, 400), (300, 400), (2600, 1100), (300, 9000), (5000, 4000)):
    x, w = torch.randn(m, 256, device="cuda").to(torch.float8_e4m3fn), torch.randn(n, 256, device="cuda").to(torch.float8_e4m3fn)
    xs, ws = torch.rand(m, 2, device="cuda"), torch.rand(-(-n // 128), 2, device="cuda")
    cases.append((edb.Fp8Weight(w, ws), x, xs, [torch.empty(m, -(-n // 16) * 16, device="cuda")[:, :n] for _ in range(4)]))
torch.cuda.synchronize()
start, failed = threading.Barrier(4), []

def work(i):
    try:
        with torch.cuda.stream(torch.cuda.Stream()):
            start.wait()
            for w, x, xs, y in cases:
                edb.mul_mat_fp8(w, x, xs, edb.make_epilogue(y[i]))
            torch.cuda.current_stream().synchronize()
    except Exception as e:
        failed.append(e)

threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
[t.start() for t in threads]
[t.join() for t in threads]
assert not failed, failed
edb.poll_status()
assert all(torch.equal(y[0], o) and bool(torch.isfinite(o).all()) for *_, y in cases for o in y)
"""


@pytest.mark.gpu
def test_first_calls_from_four_threads(edb, cuda):
    """Each kernel's first call in a process, made by four threads on streams of their own."""
    run = subprocess.run([sys.executable, "-c", FIRST_CALLS, os.path.dirname(os.path.abspath(__file__))], capture_output=True,
                         text=True, timeout=300)
    assert run.returncode == 0, run.stderr[-2000:]
