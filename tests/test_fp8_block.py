"""Block-128 e4m3 operators (edb200_quantize_fp8, edb200_mul_mat_fp8, edb200_block_norm, edb200_rope_apply) against
plain 64-bit forms, and their refusals.

Tolerances, in units of a type's rounding u (half a step relative to the value: f32 2^-24, f16 2^-11, bf16 2^-8, e4m3
2^-4, or 2^-10 of the scale among the subnormals):
  quantize    none: scale and bytes are those of the f32 formula on IEEE hardware
  mul_mat     the tensor cores' f32 sum of a block's 128 products loses at most 128 steps of 2^-23 of sum |x w| (each
              addition truncated), a block's scale is one rounding and its addition another: 128 * 2^-23 +
              (blocks + 3) * 2^-24, times sum xs ws |x| |w|; bias, gate and residual add one u each, activations
              (slope at most 1.13) 2^-18 of the value; then the output type's rounding
  block_norm  f32 sums of h terms in a tree of depth under 40: 40 u of the norm's terms, four more roundings
  rope        the angle is off by less than 2^-21 turns' worth at 2^31, by 2^-23 below 2^20; three f32 roundings
"""
import ctypes as C
import math

import pytest
import torch

U32 = 2.0 ** -24
UNIT = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 0.0, torch.float16: 2.0 ** -25, torch.bfloat16: 0.0}   # half a subnormal step
F8 = torch.float8_e4m3fn
FLOOR = 2.0 ** -100
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def up(a, b):
    return -(-a // b) * b


def laid(x, dtype, pad=0, skew=0, fill=7.0):
    """x as a view of a larger buffer: rows `pad` values longer than 16-byte units need, starting `skew` values in."""
    rows, cols = x.shape
    ld = up(cols, 16) + pad
    buf = torch.full((rows * ld + skew + 16,), fill, device=x.device).to(dtype)
    v = buf[skew:skew + rows * ld].view(rows, ld)[:, :cols]
    v.copy_(x)
    return v


def blank(rows, cols, dtype, pad=0, skew=0, fill=7.0):
    return laid(torch.full((rows, cols), fill, device="cuda"), dtype, pad, skew, fill)


def randn(*shape, seed=0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed + 17)
    return torch.randn(*shape, generator=g, device="cuda")


def blocked(x, block_rows, dtype):
    rows, k = x.shape
    p = torch.zeros(up(rows, block_rows), up(k, 128), device=x.device, dtype=dtype)
    p[:rows, :k] = x.to(dtype)
    return p.view(p.shape[0] // block_rows, block_rows, p.shape[1] // 128, 128)


def quantize_plain(x, block_rows):
    """On the CPU, whose f32 division and product round once each."""
    rows, k = x.shape
    b = blocked(x.cpu(), block_rows, torch.float32)
    fine = torch.isfinite(b)
    a = torch.where(fine, b.abs(), 0.0).amax((1, 3)).clamp_min(FLOOR)
    top = torch.full_like(a, 448.0)
    q = torch.where(fine, b * (top / a)[:, None, :, None], float("nan")).flatten(0, 1).flatten(1)[:rows, :k]
    return q.to(F8), a / top


def wide(scale, block_rows, rows, k):
    return scale.double().repeat_interleave(128, 1)[:, :k].repeat_interleave(block_rows, 0)[:rows]


def bits(q):
    return q.contiguous().view(torch.uint8)


def margins_untouched(v, fill=7.0):
    """Everything in the view's rows beyond its columns still holds `fill`."""
    base = v._base.flatten() if v._base is not None else v.flatten()
    rows, cols = v.shape
    keep = torch.ones(base.numel(), dtype=torch.bool, device=base.device)
    at = v.storage_offset() + torch.arange(rows, device=base.device)[:, None] * v.stride(0) + torch.arange(cols, device=base.device)
    keep[at.flatten()] = False
    return bool((base.float()[keep] == torch.tensor(fill).to(v.dtype).float().item()).all())


# ------------------------------------------------------------------------------------------------------- refusals
def refused(edb, status, text, code=1):
    assert status == code, (status, edb.lib().edb200_last_error())
    assert text.encode() in edb.lib().edb200_last_error()


def test_quantize_refusals(edb):
    f = edb.lib().edb200_quantize_fp8
    p = 4096     # an address that is never read: the checks come first
    for args, text in (
        ((p, edb.TYPE_Q8_0, 128, 4, 128, 1, p, 128, p, 1), "x_dtype"),
        ((p, edb.TYPE_F32, 128, 4, 128, 64, p, 128, p, 1), "block_rows"),
        ((p, edb.TYPE_F32, 128, -1, 128, 1, p, 128, p, 1), "rows"),
        ((p, edb.TYPE_F32, 128, 4, 0, 1, p, 128, p, 1), "rows"),
        ((None, edb.TYPE_F32, 128, 4, 128, 1, p, 128, p, 1), "null"),
        ((p, edb.TYPE_F32, 128, 4, 128, 1, None, 128, p, 1), "null"),
        ((p, edb.TYPE_F32, 127, 4, 128, 1, p, 128, p, 1), "ldx"),
        ((p, edb.TYPE_F32, 128, 4, 128, 1, p, 127, p, 1), "ldx"),
        ((p, edb.TYPE_F32, 129, 4, 129, 1, p, 129, p, 1), "ldx"),
        ((p + 1, edb.TYPE_F16, 128, 4, 128, 1, p, 128, p, 1), "aligned"),
        ((p, edb.TYPE_F16, 128, 4, 128, 1, p, 128, p + 2, 1), "aligned"),
    ):
        refused(edb, f(*args, None), text)
    assert f(None, edb.TYPE_F32, 128, 0, 128, 1, None, 128, None, 1, None) == edb.OK


def weight(edb, **kw):
    d = dict(w=4096, scale=4096, n=256, k=256, ldw=256, ld_scale=2)
    d.update(kw)
    return edb.Fp8WeightDesc(**d)


def epilogue(edb, **kw):
    ep = edb.Epilogue()
    ep.out, ep.out_dtype, ep.ldo = 4096, edb.TYPE_F16, 256
    for k, v in kw.items():
        setattr(ep, k, v)
    return ep


def test_mul_mat_refusals(edb):
    f = edb.lib().edb200_mul_mat_fp8

    def call(w=None, ep=None, x=4096, xs=4096, m=4, ldx=256, ld_xs=2, os=None, ld_os=0):
        return f(C.byref(w or weight(edb)), x, xs, m, ldx, ld_xs, C.byref(ep or epilogue(edb)), os, ld_os, None)

    refused(edb, f(None, 4096, 4096, 4, 256, 2, C.byref(epilogue(edb)), None, 0, None), "null")
    refused(edb, call(m=-1), "m >= 0")
    refused(edb, call(w=weight(edb, n=0)), "n >= 1")
    refused(edb, call(w=weight(edb, k=0)), "k >= 1")
    refused(edb, call(w=weight(edb, w=None)), "null")
    refused(edb, call(x=None), "null")
    refused(edb, call(xs=None), "null")
    refused(edb, call(ep=epilogue(edb, out=None)), "null")
    refused(edb, call(ldx=255), "rows of x and w")
    refused(edb, call(ldx=264), "rows of x and w")
    refused(edb, call(x=4104), "rows of x and w")
    refused(edb, call(w=weight(edb, ldw=248)), "rows of x and w")
    refused(edb, call(w=weight(edb, w=4097)), "rows of x and w")
    refused(edb, call(ld_xs=1), "scale rows")
    refused(edb, call(w=weight(edb, ld_scale=1)), "scale rows")
    refused(edb, call(ep=epilogue(edb, ldo=250)), "out rows")
    refused(edb, call(ep=epilogue(edb, ldo=260)), "out rows")
    refused(edb, call(ep=epilogue(edb, out=4098)), "out rows")
    refused(edb, call(ep=epilogue(edb, act=9)), "bad act")
    refused(edb, call(ep=epilogue(edb, out_dtype=edb.TYPE_I8)), "out_dtype")
    refused(edb, call(ep=epilogue(edb, split_n=128)), "split_n", 2)
    refused(edb, call(ep=epilogue(edb, split_k=1)), "split_k", 2)
    refused(edb, call(ep=epilogue(edb, pack=4096)), "pack", 2)
    refused(edb, call(ep=epilogue(edb, bias=4097)), "bias")
    refused(edb, call(ep=epilogue(edb, gate=4096)), "gated")
    refused(edb, call(ep=epilogue(edb, gate=4096, out_dtype=edb.TYPE_F32)), "gated")
    refused(edb, call(ep=epilogue(edb, gate=4096, out_dtype=edb.TYPE_F32, residual=4096, ld_res=258)), "gated")
    refused(edb, call(ep=epilogue(edb, gate=4096, out_dtype=edb.TYPE_F32, residual=4096, ld_res=260)), "residual's place")
    refused(edb, call(ep=epilogue(edb, out_dtype=edb.TYPE_F8_E4M3)), "out_scale")
    refused(edb, call(os=4096, ld_os=2), "out_scale")
    refused(edb, call(ep=epilogue(edb, out_dtype=edb.TYPE_F8_E4M3), os=4096, ld_os=1), "out_scale")
    assert call(m=0, x=None, xs=None) == edb.OK


def test_block_norm_refusals(edb):
    f = edb.lib().edb200_block_norm

    def call(**kw):
        d = edb.BlockNormDesc()
        base = dict(rows=4, h=256, residual=4096, ld_res=256, y=8192, ldy=256, stream_dtype=edb.TYPE_F32)
        base.update(kw)
        for k, v in base.items():
            setattr(d, k, v)
        return f(C.byref(d), None)

    refused(edb, f(None, None), "null")
    refused(edb, call(rows=-1), "rows")
    refused(edb, call(h=0), "h >= 1")
    refused(edb, call(h=16385, ld_res=20000, ldy=20000), "16384", 2)
    refused(edb, call(residual=None), "residual")
    refused(edb, call(y=None), "residual")
    refused(edb, call(post_norm=3), "EDB200_NORM")
    refused(edb, call(pre_norm=-1), "EDB200_NORM")
    refused(edb, call(stream_dtype=edb.TYPE_F8_E4M3), "types")
    refused(edb, call(x=4096, ldx=256, x_dtype=edb.TYPE_Q8_0), "types")
    refused(edb, call(z=4096, ldz=256, z_dtype=edb.TYPE_I8), "types")
    refused(edb, call(ld_res=255), "strides")
    refused(edb, call(ldy=255), "strides")
    refused(edb, call(x=4096, ldx=100), "strides")
    refused(edb, call(z=4096, ldz=100, z_dtype=edb.TYPE_F16), "strides")
    refused(edb, call(gate=4096, rows_per_mod=1, ld_mod=255), "strides")
    refused(edb, call(rows_per_mod=-1), "rows_per_mod")
    refused(edb, call(z=4096, ldz=256, z_dtype=edb.TYPE_F8_E4M3), "z_scale")
    refused(edb, call(z=4096, ldz=256, z_dtype=edb.TYPE_F8_E4M3, z_scale=4096, ld_z_scale=1), "z_scale")
    refused(edb, call(residual=4097), "aligned")
    refused(edb, call(gate=4098), "aligned")
    refused(edb, call(y=4096, ldy=264), "alias")
    assert call(rows=0, residual=None, y=None) == edb.OK


def test_rope_refusals(edb):
    for kw, text, code in (
        (dict(axes_dim=[63]), "even", 1), (dict(axes_dim=[0]), "even", 1), (dict(axes_dim=[258]), "256", 2),
        (dict(axes_dim=[64], layout=2), "layout", 1), (dict(axes_dim=[64], scaling=4), "scaling", 1),
        (dict(axes_dim=[64], theta=1.0), "theta", 1), (dict(axes_dim=[64], theta=float("nan")), "theta", 1),
        (dict(axes_dim=[64], scaling=1, factor=0.0), "factor", 1),
        (dict(axes_dim=[64], scaling=3, factor=0.5, original_length=10), "factor", 1),
        (dict(axes_dim=[64], scaling=3, factor=2.0), "original_length", 1),
        (dict(axes_dim=[64], scaling=3, factor=2.0, original_length=10, beta_fast=1.0, beta_slow=2.0), "beta", 1),
        (dict(axes_dim=[64], attention_factor=-1.0), "attention_factor", 1),
    ):
        with pytest.raises(edb.EdbError, match=text) as e:
            edb.Rope(**kw)
        assert e.value.status == code
    with pytest.raises(ValueError):
        edb.Rope([16] * 5)
    r = edb.Rope([64])
    f = edb.lib().edb200_rope_apply

    def call(q=None, k=None, dtype=edb.TYPE_F16, d=64, tokens=4, positions=None):
        base = dict(in_=4096, out=8192, in_token=256, in_head=64, out_token=256, out_head=64, heads=4)
        base.update(q or {})
        t = edb.RopeTensor(**base)
        kk = edb.RopeTensor(**{**base, **k}) if k is not None else None
        return f(r.handle, C.byref(t), C.byref(kk) if kk is not None else None, dtype, d, tokens, positions, 0, None)

    refused(edb, f(None, None, None, edb.TYPE_F16, 64, 4, None, 0, None), "null")
    refused(edb, call(dtype=edb.TYPE_I8), "dtype")
    refused(edb, call(d=62), "d_head")
    refused(edb, call(tokens=-1), "tokens")
    refused(edb, call(q=dict(out=None)), "in and out")
    refused(edb, call(q=dict(heads=0)), "in and out")
    refused(edb, call(q=dict(in_=4097)), "aligned")
    refused(edb, call(q=dict(in_token=63)), "strides")
    refused(edb, call(k=dict(out_head=32)), "strides")
    refused(edb, call(q=dict(out=4096, out_token=512)), "in place")
    refused(edb, call(positions=4098), "positions")
    assert call(tokens=0, q=dict(in_=None)) == edb.OK


@pytest.mark.gpu
def test_binding_refusals(edb, cuda):
    """What the binding sees before the library: shapes, types, strides, places."""
    t = lambda *s, dt=torch.float32: torch.zeros(*s, device="cuda", dtype=dt)  # noqa: E731
    x, q, s = t(4, 256), t(4, 256, dt=F8), t(4, 2)
    for bad in (dict(x=x.cpu()), dict(q=t(4, 255, dt=F8)), dict(q=t(4, 256)), dict(scale=t(4, 3)), dict(scale=t(4, 2, dt=torch.float16)),
                dict(x=t(256, 4).t()), dict(block_rows=64)):
        with pytest.raises(ValueError):
            edb.quantize_fp8(**{**dict(x=x, q=q, scale=s), **bad})
    with pytest.raises(edb.EdbError):                        # one row for all of them: no stride
        edb.quantize_fp8(t(1, 256).expand(4, 256), q, s)
    with pytest.raises(ValueError):
        edb.Fp8Weight(t(128, 256, dt=F8), t(2, 2))
    w = edb.Fp8Weight(t(128, 256, dt=F8), t(1, 2))
    ep = edb.make_epilogue(t(4, 128))
    for bad in (dict(x=t(4, 240, dt=F8)), dict(x=x), dict(x_scale=t(4, 1)), dict(out_scale=t(4, 2)), dict(x_scale=s.cpu())):
        with pytest.raises(ValueError):
            edb.mul_mat_fp8(**{**dict(w=w, x=q, x_scale=s, ep=ep), **bad})
    r, y = t(4, 256), t(4, 256)
    for bad in (dict(y=t(4, 255)), dict(y=t(4, 256, dt=torch.float16)), dict(x=t(3, 256)), dict(z=t(4, 128)), dict(z_scale=t(4, 1)),
                dict(gate=t(255)), dict(gate=t(256, dt=torch.float16)), dict(gate=t(1, 256), rows_per_mod=2), dict(post_weight=t(255)),
                dict(gate=t(1, 256).expand(4, 256), scale=t(4, 256), rows_per_mod=1), dict(pre_bias=t(512)[::2]),
                dict(scale=t(4, 256), shift=t(4, 260)[:, :256], rows_per_mod=1), dict(gate=t(256).cpu())):
        with pytest.raises(ValueError):
            edb.block_norm(**{**dict(residual=r, y=y), **bad})
    with pytest.raises(edb.EdbError):
        edb.block_norm(r, y, x=r, gate=t(1, 256).expand(4, 256), rows_per_mod=1)
    rope, a = edb.Rope([64]), t(4, 2, 64)
    pos = torch.zeros(4, 1, device="cuda", dtype=torch.int32)
    for bad in (dict(q_out=t(4, 2, 63)), dict(q_out=t(4, 2, 64, dt=torch.float16)), dict(positions=pos.long()), dict(positions=pos[:3]),
                dict(k=t(3, 2, 64), k_out=t(3, 2, 64)), dict(q=t(4, 64, 2).transpose(1, 2)), dict(positions=pos.cpu())):
        with pytest.raises(ValueError):
            rope.apply(**{**dict(positions=pos, q=a, q_out=a), **bad})


@pytest.mark.gpu
def test_nothing_to_do(edb, cuda):
    """No rows, no tokens: nothing is read, written or launched."""
    t = lambda *s, dt=torch.float32: torch.zeros(*s, device="cuda", dtype=dt)  # noqa: E731
    n0 = edb.lib().edb200_launch_count()
    edb.quantize_fp8(t(0, 256), t(0, 256, dt=F8), t(0, 2))
    edb.mul_mat_fp8(edb.Fp8Weight(t(128, 256, dt=F8), t(1, 2)), t(0, 256, dt=F8), t(0, 2), edb.make_epilogue(t(0, 128)))
    edb.block_norm(t(0, 256), t(0, 256))
    edb.Rope([64]).apply(None, t(0, 2, 64), t(0, 2, 64))
    assert edb.lib().edb200_launch_count() == n0


# ------------------------------------------------------------------------------------------------------- quantize
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,k,block_rows,pad,skew", [
    (1, 1, 1, 0, 0), (1, 127, 1, 0, 0), (3, 128, 1, 0, 0), (5, 129, 1, 3, 1), (33, 1000, 1, 0, 0), (7, 5120, 1, 16, 0),
    (1, 130, 128, 0, 0), (127, 128, 128, 0, 0), (128, 256, 128, 0, 0), (300, 200, 128, 16, 0), (129, 77, 128, 5, 3)])
def test_quantize(edb, cuda, dtype, rows, k, block_rows, pad, skew):
    x = laid(randn(rows, k, seed=rows + k) * torch.exp(4 * randn(rows, 1, seed=k)), dtype, pad, skew)
    q, s = blank(rows, k, F8, pad, skew), blank(-(-rows // block_rows), -(-k // 128), torch.float32, 1)
    edb.quantize_fp8(x, q, s, block_rows)
    want_q, want_s = quantize_plain(x, block_rows)
    assert torch.equal(s.cpu(), want_s)
    fine = torch.isfinite(x)        # rows this strong reach infinity in f16: NaN, of which there are two bytes
    assert torch.equal(bits(q)[fine].cpu(), bits(want_q)[fine.cpu()]) and torch.equal(torch.isnan(q.float()), ~fine)
    assert margins_untouched(q) and margins_untouched(s)
    # the definition in 64 bits: each value within half a step of e4m3, three f32 roundings besides
    w, x64 = wide(s, block_rows, rows, k), x.double()
    step = torch.maximum(x64.abs() * 2.0 ** -4, w * 2.0 ** -10)
    assert bool(((q.double() * w - x64).abs() <= step * (1 + 2.0 ** -15) + x64.abs() * 4 * U32)[fine].all())


@pytest.mark.gpu
def test_quantize_rows_of_many_blocks(edb, cuda):
    """So many blocks a row that a block's row is found by division in 64 bits: 11 x 20001 blocks."""
    rows, k = 11, 20000 * 128 + 5
    x = laid(randn(rows, k, seed=5), torch.float16)
    q, s = blank(rows, k, F8), blank(rows, 20001, torch.float32, 1)
    edb.quantize_fp8(x, q, s)
    want_q, want_s = quantize_plain(x, 1)
    assert torch.equal(bits(q.cpu()), bits(want_q)) and torch.equal(s.cpu(), want_s)
    assert margins_untouched(q) and margins_untouched(s)


@pytest.mark.gpu
@pytest.mark.parametrize("block_rows", [1, 128])
def test_quantize_extremes(edb, cuda, block_rows):
    """Zero blocks, tiny and huge magnitudes, values that are not finite: only those become NaN."""
    x = torch.zeros(256, 512, device="cuda")
    x[0, 0], x[0, 1] = 2.0 ** -149, -(2.0 ** -140)
    x[1, 130], x[1, 131] = 3.4e38, -1e30
    x[2, 256], x[2, 257], x[2, 258], x[2, 259] = float("inf"), float("-inf"), float("nan"), 3.0
    x[130] = float("nan")
    x[131, 5] = 1e-30
    q, s = torch.empty(256, 512, device="cuda", dtype=F8), torch.empty(256 // block_rows, 4, device="cuda")
    edb.quantize_fp8(x, q, s, block_rows)
    want_q, want_s = quantize_plain(x, block_rows)
    assert torch.equal(s.cpu(), want_s) and bool((s > 0).all())
    same = bits(q.cpu()) == bits(want_q)
    both_nan = torch.isnan(q.float().cpu()) & torch.isnan(want_q.float())   # NaN has two bytes
    assert bool((same | both_nan).all())
    assert torch.equal(torch.isnan(q.float()), ~torch.isfinite(x))


# -------------------------------------------------------------------------------------------------------- mul_mat
def fp8_operand(rows, k, block_rows, seed, pad=0, size=1.0):
    x = randn(rows, k, seed=seed) * size * torch.exp(randn(rows, 1, seed=seed + 1))
    q, s = quantize_plain(x, block_rows)
    return laid(q.float().cuda(), F8, pad), s.cuda()


ACTS = {"none": 0, "gelu_tanh": 1, "silu": 2, "gelu_erf": 3}


def act64(y, act):
    if act == "gelu_tanh":
        return 0.5 * y * (1 + torch.tanh(math.sqrt(2 / math.pi) * (y + 0.044715 * y ** 3)))
    if act == "gelu_erf":
        return 0.5 * y * (1 + torch.erf(y / math.sqrt(2)))
    return y * torch.sigmoid(y) if act == "silu" else y


def linear64(xq, xs, wq, ws, bias, act):
    """Value and error bound before the output's own rounding."""
    m, k = xq.shape
    n = wq.shape[0]
    x, w = xq.double() * wide(xs, 1, m, k), wq.double() * wide(ws, 128, n, k)
    y, size = x @ w.t(), x.abs() @ w.abs().t()
    err = size * (128 * 2.0 ** -23 + (-(-k // 128) + 3) * U32)
    if bias is not None:
        y = y + bias.double()
        err = err + y.abs() * U32
    z = act64(y, act)
    if act != "none":
        err = 1.13 * err + z.abs() * 2.0 ** -18 + y.abs() * 2.0 ** -23
    return z, err


def run_linear(edb, m, k, n, out, act="none", bias=True, pad=0, seed=0, in_place=False):
    xq, xs = fp8_operand(m, k, 1, seed, pad)
    wq, ws = fp8_operand(n, k, 128, seed + 5, pad, 0.05)
    b = randn(n, seed=seed + 9) if bias else None
    want, err = linear64(xq, xs, wq, ws, b, act)
    dtype = {"gated": torch.float32, "f8": F8}.get(out, out)
    y = blank(m, n, dtype, pad)
    ys = blank(m, -(-n // 128), torch.float32, 1) if out == "f8" else None
    res = gate = None
    if out == "gated":
        res, gate = laid(3 * randn(m, n, seed=seed + 11), torch.float32, pad), randn(n, seed=seed + 12)
        want, err = res.double() + gate.double() * want, gate.double().abs() * err
        err = err + (res.double().abs() + want.abs()) * 2 * U32
        if in_place:
            y.copy_(res)
            res = y
    ep = edb.make_epilogue(y, bias=b, act=ACTS[act], residual=res, gate=gate)
    edb.mul_mat_fp8(edb.Fp8Weight(wq, ws), xq, xs, ep, ys)
    edb.poll_status()
    if out == "f8":
        # the scale is the row block's maximum / 448, each value within half a step of it
        top = blocked(want, 1, torch.float64).abs().amax((1, 3)).clamp_min(FLOOR)
        room = blocked(err, 1, torch.float64).amax((1, 3))
        assert bool(((ys.double() * 448 - top).abs() <= room + top * 4 * U32).all())
        w = wide(ys, 1, m, n)
        step = torch.maximum((want.abs() + err) * 2.0 ** -4, w * 2.0 ** -10) * (1 + 2.0 ** -10)
        assert bool(((y.double() * w - want).abs() <= err + step + want.abs() * 4 * U32).all())
        assert margins_untouched(ys)
    else:
        off = (y.double() - want).abs()
        room = err + (want.abs() + err) * UNIT[dtype] + TINY[dtype]
        worst = (off / room).max().item()
        assert worst <= 1.0, worst
    if not in_place:
        assert margins_untouched(y)
    return y


SHAPES = [(1, 1, 1), (1, 16, 128), (2, 128, 130), (5, 129, 257), (8, 5120, 640), (17, 1000, 96), (33, 256, 300),
          (64, 2048, 512), (77, 384, 1536), (100, 4224, 129), (129, 640, 384), (200, 1536, 1000), (257, 72, 255),
          (513, 512, 513), (1024, 3584, 768)]


@pytest.mark.gpu
@pytest.mark.parametrize("m,k,n", SHAPES)
@pytest.mark.parametrize("out", [torch.float32, torch.float16, "gated", "f8"])
def test_mul_mat(edb, cuda, m, k, n, out):
    run_linear(edb, m, k, n, out, act="gelu_tanh" if out == "f8" else "none", pad=16 if m % 2 else 0, seed=m + k + n)


@pytest.mark.gpu
@pytest.mark.parametrize("m,k,n", [(3, 300, 260), (70, 300, 260), (150, 700, 520)])
@pytest.mark.parametrize("act", sorted(ACTS))
@pytest.mark.parametrize("bias", [True, False])
@pytest.mark.parametrize("out", [torch.bfloat16, torch.float32])
def test_mul_mat_epilogues(edb, cuda, m, k, n, act, bias, out):
    run_linear(edb, m, k, n, out, act=act, bias=bias, seed=k)


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 40, 300])
def test_mul_mat_residual_in_place(edb, cuda, m):
    run_linear(edb, m, 512, 384, "gated", in_place=True, pad=16)


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 7, 60, 140, 700])
def test_mul_mat_is_the_same_every_run_and_row_by_row(edb, cuda, m):
    """The same bits again, and a NaN row or scale stays in its row."""
    k, n = 640, 300
    xq, xs = fp8_operand(m, k, 1, 3)
    wq, ws = fp8_operand(n, k, 128, 4)
    w = edb.Fp8Weight(wq, ws)

    def run():
        y = torch.empty(m, 304, device="cuda")[:, :n]
        edb.mul_mat_fp8(w, xq, xs, edb.make_epilogue(y))
        return y.clone()

    first = run()
    assert torch.equal(first, run())
    bad = m // 2
    xs[bad, 1] = float("nan")
    if m > 1:
        xq[0, 5] = float("nan")
    got = run()
    rows = torch.zeros(m, dtype=torch.bool, device="cuda")
    rows[bad] = True
    rows[0] = True if m > 1 else rows[0]
    assert bool(torch.isnan(got[rows]).all())
    assert torch.equal(got[~rows], first[~rows])


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 20, 150, 600])
def test_mul_mat_quantised_output_of_rows_not_finite(edb, cuda, m):
    """An infinity in a row's activated block reaches the next product as NaN, and its neighbours keep their scale."""
    k, n = 256, 260
    xq, xs = fp8_operand(m, k, 1, 3)
    wq, ws = fp8_operand(n, k, 128, 4)
    bias = torch.zeros(n, device="cuda")
    bias[3] = float("inf")
    y, ys = blank(m, n, F8), torch.empty(m, 3, device="cuda")
    edb.mul_mat_fp8(edb.Fp8Weight(wq, ws), xq, xs, edb.make_epilogue(y, bias=bias), ys)
    plain, _ = linear64(xq, xs, wq, ws, None, "none")
    assert torch.equal(torch.isnan(y.float()), torch.isinf(bias)[None].expand(m, n))
    plain[:, 3] = 0.0
    top = blocked(plain, 1, torch.float64).abs().amax((1, 3))
    assert bool(((ys.double() * 448 - top).abs() <= top * 2.0 ** -12).all())


@pytest.mark.gpu
@pytest.mark.parametrize("m,k,n", [(2, 12800, 256), (40, 9000, 130), (130, 20480, 200), (200, 1400, 300), (600, 2304, 5300),
                                   (2600, 500, 2100), (19000, 130, 260)])
def test_mul_mat_long_sums_and_many_tiles(edb, cuda, m, k, n):
    """k split over clusters, groups of eight blocks that end early, tiles walked by resident CTA pairs in chunks."""
    run_linear(edb, m, k, n, torch.float32, seed=k)
    run_linear(edb, m, k, n, "f8", act="silu", seed=k + 1)


@pytest.mark.gpu
def test_offsets_beyond_32_bits(edb, cuda):
    """Rows so far apart that a row's offset passes 2^32 bytes and 2^31 elements."""
    far, rows, k = (1 << 30) + 64, 3, 256
    big = torch.empty(2 * far + 4096, device="cuda", dtype=torch.float16)
    x = big.as_strided((rows, k), (far, 1))
    x.copy_(randn(rows, k, seed=3))
    q, s = torch.empty(rows, k, device="cuda", dtype=F8), torch.empty(rows, 2, device="cuda")
    edb.quantize_fp8(x, q, s)
    want_q, want_s = quantize_plain(x.contiguous(), 1)
    assert torch.equal(bits(q.cpu()), bits(want_q)) and torch.equal(s.cpu(), want_s)
    wq, ws = fp8_operand(n := 384, k, 128, 7, 0, 0.05)
    want, err = linear64(q, s, wq, ws, None, "none")
    y = big.as_strided((rows, n), (far, 1), 512)
    edb.mul_mat_fp8(edb.Fp8Weight(wq, ws), q, s, edb.make_epilogue(y))
    assert bool(((y.double() - want).abs() <= err + (want.abs() + err) * UNIT[torch.float16] + TINY[torch.float16]).all())
    z = big.as_strided((rows, k), (far, 1), 1024)
    edb.block_norm(x, z, None, residual_scale=2.0)
    assert torch.equal(z, x * 2)
    t = big.as_strided((rows, 2, 128), (far, 128, 1), 2048)
    edb.Rope([128]).apply(None, x.unflatten(1, (2, 128)), t)
    assert torch.equal(t[0].flatten(), x[0])
    small = torch.empty(rows, 2, 128, device="cuda", dtype=torch.float16)
    edb.Rope([128]).apply(None, x.contiguous().unflatten(1, (2, 128)), small)
    assert torch.equal(t, small)


@pytest.mark.gpu
def test_two_streams_and_two_recordings_at_once(edb, cuda):
    """No call keeps anything outside its arguments: the same products from two streams, eager and recorded, side by side."""
    m, k, n = 300, 1280, 1100
    xq, xs = fp8_operand(m, k, 1, 1)
    wq, ws = fp8_operand(n, k, 128, 2, 0, 0.05)
    w = edb.Fp8Weight(wq, ws)
    outs = [torch.empty(m, 1104, device="cuda")[:, :n] for _ in range(5)]
    edb.mul_mat_fp8(w, xq, xs, edb.make_epilogue(outs[4]))
    torch.cuda.synchronize()
    streams, graphs = [torch.cuda.Stream(), torch.cuda.Stream()], []
    for i, st in enumerate(streams):
        with torch.cuda.stream(st):
            graphs.append(edb.Graph(lambda i=i: edb.mul_mat_fp8(w, xq, xs, edb.make_epilogue(outs[i]))))
    for _ in range(20):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                graphs[i].launch()
                edb.mul_mat_fp8(w, xq, xs, edb.make_epilogue(outs[2 + i]))
    torch.cuda.synchronize()
    edb.poll_status()
    for o in outs[:4]:
        assert torch.equal(o, outs[4])


# ----------------------------------------------------------------------------------------------------- block_norm
def norm64(v, kind, w, b, eps):
    """Value and a bound on the f32 error, in units of U32."""
    if kind == 0:
        return v, torch.zeros_like(v)
    h = v.shape[1]
    mean = v.mean(1, keepdim=True) if kind == 1 else 0.0
    c = v - mean
    r = 1 / torch.sqrt((c * c).mean(1, keepdim=True) + eps)
    spread = v.abs().mean(1, keepdim=True) if kind == 1 else 0.0
    out = c * r
    err = (40 * (c.abs() + spread) + 4 * v.abs()) * r
    if w is not None:
        out, err = out * w.double(), err * w.double().abs()
    if b is not None:
        out = out + b.double()
    return out, err + 3 * out.abs()


def run_norm(edb, rows, h, x_dtype, s_dtype, z, post, pre, rpm=0, pad=0, skew=0, affine=True, x=True, y=True, mod=True, in_place=None):
    xv = laid(randn(rows, h, seed=1) * torch.exp(randn(rows, 1, seed=2)) + 0.5, x_dtype, pad, skew) if x else None
    rv = laid(3 * randn(rows, h, seed=3) - 1.0, s_dtype, pad, skew)
    groups = -(-rows // rpm) if rpm else 1
    g, sc, sh = (laid(0.5 * randn(groups, h, seed=4 + i), torch.float32, pad, skew) if mod else None for i in range(3))
    aff = [1 + 0.2 * randn(h, seed=8 + i) if affine else None for i in range(4)]
    eps, rs = 1e-5, 0.75
    # the plain form
    which = torch.arange(rows, device="cuda") // rpm if rpm else torch.zeros(rows, dtype=torch.int64, device="cuda")
    y64, e = rs * rv.double(), 2 * (rs * rv.double()).abs()
    if x:
        t, te = norm64(xv.double(), post, aff[0] if post else None, aff[1] if post else None, eps)
        gg = g.double()[which] if mod else 1.0
        y64 = y64 + gg * t
        e = e + te * abs(gg) + (gg * t).abs() + y64.abs()
    z64, ze = norm64(y64, pre, aff[2] if pre else None, aff[3] if pre else None, eps)
    if pre:   # what y's error does to z
        c = y64 - (y64.mean(1, keepdim=True) if pre == 1 else 0.0)
        r = 1 / torch.sqrt((c * c).mean(1, keepdim=True) + eps)
        rms = torch.sqrt((e * e).mean(1, keepdim=True))
        carried = (e + rms * (1 + (c * r).abs())) * r
        ze = ze + carried * (aff[2].double().abs() if aff[2] is not None else 1.0)
    else:
        ze = ze + e
    if mod:
        m = 1 + sc.double()[which]
        ze = ze * m.abs() + 2 * (z64 * m).abs() + 2 * z64.abs()
        z64 = z64 * m + sh.double()[which]
        ze = ze + z64.abs()
    # the call
    z_dtype = F8 if z == "f8" else z
    yv = blank(rows, h, s_dtype, pad, skew) if y else None
    if in_place == "residual":
        yv = rv
    elif in_place == "x":
        yv = xv
    zv = blank(rows, h, z_dtype, pad, skew) if z is not None else None
    zs = blank(rows, -(-h // 128), torch.float32, 1) if z == "f8" else None
    edb.block_norm(rv, yv, zv, zs, x=xv, gate=g if x else None, residual_scale=rs, post_norm=post,
                   post_weight=aff[0] if post else None, post_bias=aff[1] if post else None, post_eps=eps, pre_norm=pre,
                   pre_weight=aff[2] if pre else None, pre_bias=aff[3] if pre else None, pre_eps=eps, scale=sc, shift=sh,
                   rows_per_mod=rpm)
    if yv is not None:
        room = e * U32 + (y64.abs() + e * U32) * UNIT[s_dtype] + TINY[s_dtype]
        assert bool(((yv.double() - y64).abs() <= room).all())
        assert in_place or margins_untouched(yv)
    if z == "f8":
        top = blocked(z64, 1, torch.float64).abs().amax((1, 3)).clamp_min(FLOOR)
        room = blocked(ze, 1, torch.float64).amax((1, 3)) * U32
        assert bool(((zs.double() * 448 - top).abs() <= room + top * 4 * U32).all())
        w = wide(zs, 1, rows, h)
        step = torch.maximum((z64.abs() + ze * U32) * 2.0 ** -4, w * 2.0 ** -10) * (1 + 2.0 ** -10)
        assert bool(((zv.double() * w - z64).abs() <= ze * U32 + step + z64.abs() * 4 * U32).all())
        assert margins_untouched(zs)
    elif z is not None:
        room = ze * U32 + (z64.abs() + ze * U32) * UNIT[z_dtype] + TINY[z_dtype]
        assert bool(((zv.double() - z64).abs() <= room).all())
    assert zv is None or margins_untouched(zv)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,h,rpm,pad,skew", [
    (1, 1, 0, 0, 0), (3, 7, 1, 0, 0), (9, 64, 4, 0, 0), (17, 255, 5, 0, 0), (8, 256, 0, 0, 0), (5, 264, 2, 8, 0),
    (4, 1000, 1, 0, 0), (6, 1024, 3, 0, 0), (3, 1032, 0, 0, 0), (154, 1536, 77, 0, 0), (5, 2049, 2, 3, 1), (2, 5120, 1, 16, 0),
    (3, 8200, 0, 0, 0), (2, 16384, 1, 0, 0)])
@pytest.mark.parametrize("post,pre,z", [(0, 1, torch.float16), (2, 2, "f8"), (1, 0, torch.bfloat16), (2, 1, torch.float32)])
def test_block_norm(edb, cuda, rows, h, rpm, pad, skew, post, pre, z):
    run_norm(edb, rows, h, torch.bfloat16, torch.float32, z, post, pre, rpm, pad, skew)


@pytest.mark.gpu
@pytest.mark.parametrize("h", [200, 1600])
@pytest.mark.parametrize("x_dtype", DTYPES)
@pytest.mark.parametrize("s_dtype", DTYPES)
@pytest.mark.parametrize("z", [torch.float32, torch.float16, torch.bfloat16, "f8"])
def test_block_norm_types(edb, cuda, h, x_dtype, s_dtype, z):
    run_norm(edb, 21, h, x_dtype, s_dtype, z, 2, 1, 4)


@pytest.mark.gpu
@pytest.mark.parametrize("h", [96, 1280])
def test_block_norm_parts(edb, cuda, h):
    """Each operand left out in turn, and y in the place of the residual or of x."""
    kw = dict(rows=11, h=h, x_dtype=torch.float32, s_dtype=torch.float32)
    run_norm(edb, z="f8", post=0, pre=2, x=False, **kw)
    run_norm(edb, z=torch.float16, post=0, pre=1, x=False, y=False, **kw)
    run_norm(edb, z=None, post=2, pre=0, **kw)
    run_norm(edb, z=torch.float16, post=2, pre=2, affine=False, mod=False, **kw)
    run_norm(edb, z="f8", post=1, pre=2, y=False, **kw)
    run_norm(edb, z="f8", post=2, pre=2, in_place="residual", **kw)
    run_norm(edb, z=torch.float16, post=2, pre=2, in_place="x", **kw)


@pytest.mark.gpu
def test_block_norm_rows_stay_apart(edb, cuda):
    """A row of NaN, of infinities or of zeros changes no other row."""
    for h in (160, 1664):
        x, r = randn(9, h, seed=1), randn(9, h, seed=2)
        out = []
        for poison in (False, True):
            if poison:
                x[2], r[4], x[6], r[6] = float("nan"), float("inf"), 0.0, 0.0
            y, z, s = torch.empty_like(r), torch.empty(9, h, device="cuda", dtype=F8), torch.empty(9, -(-h // 128), device="cuda")
            edb.block_norm(r, y, z, s, x=x, post_norm=edb.NORM_RMS, pre_norm=edb.NORM_LAYER)
            out.append((y, bits(z), s))
        keep = [0, 1, 3, 5, 7, 8]
        for a, b in zip(*out):
            assert torch.equal(a[keep], b[keep])
        y, z, s = out[1]
        assert bool(torch.isnan(y[2]).all()) and bool(torch.isnan(z.view(F8).float()[[2, 4]]).all())
        assert bool((y[6] == 0).all()) and bool((z.view(F8).float()[6] == 0).all()) and bool(torch.isfinite(s).all())


# ----------------------------------------------------------------------------------------------------------- rope
def rope_pairs(axes, scaling, factor, theta, original):
    pairs = []
    for axis, dim in enumerate(axes):
        base = theta * factor ** (dim / (dim - 2)) if scaling == "ntk" and dim > 2 else theta

        def place(turns):
            return dim * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(theta))

        low, high = max(math.floor(place(32.0)), 0), min(math.ceil(place(1.0)), dim - 1)
        for j in range(dim // 2):
            f = base ** (-2.0 * j / dim)
            if scaling == "linear":
                f = f / factor
            elif scaling == "yarn":
                ramp = min(max((j - low) / max(high - low, 1e-3), 0.0), 1.0)
                f = f / factor * ramp + f * (1 - ramp)
            pairs.append((axis, f))
    return pairs, 0.1 * math.log(factor) + 1 if scaling == "yarn" else 1.0


def rope64(x, positions, pairs, mul, half, inverse):
    p = len(pairs)
    out = x.double().clone()
    for i, (axis, f) in enumerate(pairs):
        a, b = (i, i + p) if half else (2 * i, 2 * i + 1)
        t = positions[:, axis].double() * f * (-1 if inverse else 1)
        c, s = (torch.cos(t) * mul)[:, None], (torch.sin(t) * mul)[:, None]
        va, vb = x[..., a].double(), x[..., b].double()
        out[..., a], out[..., b] = va * c - vb * s, va * s + vb * c
    return out


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("tokens,hq,hk,d,axes,scaling", [
    (1, 1, 0, 2, [2], "none"), (5, 3, 1, 64, [64], "none"), (7, 2, 2, 80, [40], "linear"), (33, 24, 24, 64, [16, 24, 24], "ntk"),
    (9, 40, 8, 128, [44, 42, 42], "yarn"), (50, 1, 1, 128, [64], "yarn"), (3, 5, 0, 256, [256], "none"), (4, 2, 1, 100, [6, 4, 2, 10], "ntk"),
    (1000, 1, 1, 16, [4], "none"), (2, 200, 40, 256, [64, 64], "linear")])
def test_rope(edb, cuda, dtype, half, tokens, hq, hk, d, axes, scaling):
    factor, theta, original = 4.0, 10000.0, 300.0
    pairs, mul = rope_pairs(axes, scaling, factor, theta, original)
    r = edb.Rope(axes, theta, edb.ROPE_HALF if half else edb.ROPE_INTERLEAVED,
                 {"none": 0, "linear": 1, "ntk": 2, "yarn": 3}[scaling], factor, original)
    g = torch.Generator(device="cuda")
    g.manual_seed(tokens)
    pos = torch.randint(-(1 << 20), 1 << 20, (tokens, len(axes)), generator=g, device="cuda", dtype=torch.int32)
    both = randn(tokens, (hq + hk) * d, seed=d).to(dtype)
    q = both[:, :hq * d].view(tokens, hq, d)
    k = both[:, hq * d:].view(tokens, hk, d) if hk else None
    q_out = torch.full((hq, tokens + 1, d), 9.0, device="cuda", dtype=dtype)       # head-major, a row to spare
    k_out = torch.full((tokens, hk, d + 8), 9.0, device="cuda", dtype=dtype) if hk else None
    for inverse in (False, True):
        r.apply(pos, q, q_out.transpose(0, 1)[:tokens], k, k_out[..., :d] if hk else None, inverse)
        for got, x in ((q_out.transpose(0, 1)[:tokens], q), (k_out[..., :d], k) if hk else (None, None)):
            if got is None:
                continue
            want = rope64(x, pos, pairs, mul, half, inverse)
            # |a| + |b| of a pair is at most sqrt(2) times its size; the angle is off by 2^-21 at most at 2^20 turns
            size = x.double().abs().amax(-1, keepdim=True) * mul * 2
            room = size * (2.0 ** -22 + 6 * U32) + want.abs() * UNIT[dtype] * (1 + 2.0 ** -10) + TINY[dtype]
            assert bool(((got.double() - want).abs() <= room).all())
            assert torch.equal(got[..., sum(axes):], x[..., sum(axes):])
    assert bool((q_out[:, tokens] == 9.0).all())
    assert k_out is None or bool((k_out[..., d:] == 9.0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_rope_in_place_and_odd_places(edb, cuda, dtype):
    """In place equals out of place; unaligned strides take single values and give the same bits; no positions: the index."""
    for half in (0, 1):
        r = edb.Rope([32], layout=half)
        x = randn(37, 3, 48, seed=4).to(dtype)
        pos = torch.arange(37, device="cuda", dtype=torch.int32)[:, None].contiguous()
        want = torch.empty_like(x)
        r.apply(pos, x, want)
        y = x.clone()
        r.apply(None, y, y)
        assert torch.equal(y, want)
        odd = torch.zeros(37 * 3 * 49 + 1, device="cuda", dtype=dtype)[1:].view(37, 3, 49)[..., :48]
        odd.copy_(x)
        r.apply(pos, odd, odd)
        assert torch.equal(odd, want)
        r.apply(pos, want, want, inverse=True)
        assert bool(((want.double() - x.double()).abs() <= x.double().abs().amax() * 4 * UNIT[dtype]).all())


@pytest.mark.gpu
def test_rope_far_positions(edb, cuda):
    """The ends of the 32-bit range: the angle's 64-bit product is off by 2.4e-7 rad there."""
    r = edb.Rope([128])
    pos = torch.tensor([[2 ** 31 - 1], [-2 ** 31], [123456789], [0]], device="cuda", dtype=torch.int32)
    x = randn(4, 2, 128, seed=1)
    out = torch.empty_like(x)
    r.apply(pos, x, out)
    pairs, mul = rope_pairs([128], "none", 1.0, 10000.0, 1.0)
    want = rope64(x, pos, pairs, mul, False, False)
    # the plain form's own product rounds at 2^31 * 2^-53, too
    assert bool(((out.double() - want).abs() <= x.abs().double().amax() * 2 * (3 * 2.4e-7 + 6 * U32)).all())


@pytest.mark.gpu
def test_rope_gradient(edb, cuda):
    """inverse is the transpose of the forward call: <R x, g> = <x, R^T g>, and by differences."""
    r = edb.Rope([44, 42, 42], layout=edb.ROPE_HALF, scaling=edb.ROPE_SCALE_YARN, factor=4.0, original_length=300)
    pos = torch.randint(-500, 500, (13, 3), device="cuda", dtype=torch.int32)
    x, g = randn(13, 4, 128, seed=1), randn(13, 4, 128, seed=2)
    rx, rg = torch.empty_like(x), torch.empty_like(x)
    r.apply(pos, x, rx)
    r.apply(pos, g, rg, inverse=True)
    a, b = (rx.double() * g.double()).sum(), (x.double() * rg.double()).sum()
    assert abs(a - b) <= (rx.double() * g.double()).abs().sum() * 16 * U32
    moved = x.clone()
    moved[3, 1, 70] += 1.0                       # linear: a difference of any size is the derivative
    r.apply(pos, moved, moved)
    by_difference = ((moved.double() - rx.double()) * g.double()).sum()
    assert abs(by_difference - rg[3, 1, 70].double()) <= 64 * U32 * x.abs().amax() * g.abs().amax() * 4


# ------------------------------------------------------------------------------------------- as they are used together
@pytest.mark.gpu
def test_one_block_round(edb, cuda):
    """norm -> fp8 q, k, v -> rope head-major -> attention -> fp8 out-projection into the stream -> norm -> feed-forward,
    eager and replayed from a recording on another stream, against the same round in 64 bits."""
    t, heads, d, ff = 150, 4, 64, 640
    h = heads * d
    gen = lambda *s, seed: randn(*s, seed=seed)  # noqa: E731
    ws = {}
    for i, (name, n, k) in enumerate((("qkv", 3 * h, h), ("out", h, h), ("up", ff, h), ("down", h, ff))):
        q, s = quantize_plain(gen(n, k, seed=40 + i) / math.sqrt(k), 128)
        ws[name] = (q.cuda(), s.cuda())
    layers = {name: edb.Fp8Weight(*w) for name, w in ws.items()}
    stream0 = gen(t, h, seed=60)
    gate, scale, shift = (0.5 * gen(h, seed=61 + i) for i in range(3))
    pos = torch.arange(t, device="cuda", dtype=torch.int32)[:, None] * 3 - 40
    rope = edb.Rope([d], layout=edb.ROPE_HALF)
    f16, f8 = torch.float16, F8
    e = lambda *s, dt=torch.float32: torch.zeros(*s, device="cuda", dtype=dt)  # noqa: E731
    b = dict(n1=e(t, h, dt=f8), n1s=e(t, 2), qkv=e(t, 3 * h, dt=f16), q=e(heads, t, d, dt=f16), k=e(heads, t, d, dt=f16),
             v=e(heads, t, d, dt=f16), att=e(t, h, dt=f16), a8=e(t, h, dt=f8), a8s=e(t, 2), x=e(t, h), n2=e(t, h, dt=f8),
             n2s=e(t, 2), up=e(t, ff, dt=f8), ups=e(t, 5), proj=e(t, h, dt=f16), y=e(t, h))

    def round_():
        edb.block_norm(stream0, None, b["n1"], b["n1s"], pre_norm=edb.NORM_LAYER, scale=scale, shift=shift)
        edb.mul_mat_fp8(layers["qkv"], b["n1"], b["n1s"], edb.make_epilogue(b["qkv"]))
        q, k, v = (b["qkv"][:, i * h:(i + 1) * h].view(t, heads, d) for i in range(3))
        rope.apply(pos, q, b["q"].transpose(0, 1), k, b["k"].transpose(0, 1))
        b["v"].copy_(v.transpose(0, 1))
        edb.check(edb.lib().edb200_attention_f16(edb.ptr(b["q"]), edb.ptr(b["k"]), edb.ptr(b["v"]), heads, t, t, d, d ** -0.5,
                                                 edb.ptr(b["att"]), edb.TYPE_F16, h, edb.current_stream()))
        edb.quantize_fp8(b["att"], b["a8"], b["a8s"])
        edb.mul_mat_fp8(layers["out"], b["a8"], b["a8s"], edb.make_epilogue(b["x"], residual=stream0, gate=gate))
        edb.block_norm(b["x"], None, b["n2"], b["n2s"], pre_norm=edb.NORM_RMS)
        edb.mul_mat_fp8(layers["up"], b["n2"], b["n2s"], edb.make_epilogue(b["up"], act=edb.ACT_GELU_TANH), b["ups"])
        edb.mul_mat_fp8(layers["down"], b["up"], b["ups"], edb.make_epilogue(b["proj"]))
        edb.block_norm(b["x"], b["y"], None, x=b["proj"], gate=gate, post_norm=edb.NORM_RMS)

    def step64(q, s, name):
        x = q.double() * wide(s, 1, *q.shape)
        w = ws[name][0].double() * wide(ws[name][1], 128, *ws[name][0].shape)
        return x @ w.t()

    def near(got, want, rel):
        return ((got.double() - want).norm() / want.norm()).item() <= rel

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        round_()
    side.synchronize()
    edb.poll_status()
    # each stage from the stage before as the kernels left it: a stage's own rounding is what is compared
    n1, _ = norm64(stream0.double(), 1, None, None, 1e-6)
    assert near(b["n1"].double() * wide(b["n1s"], 1, t, h), n1 * (1 + scale.double()) + shift.double(), 2.0 ** -4)
    qkv = step64(b["n1"], b["n1s"], "qkv")
    assert near(b["qkv"], qkv, 2.0 ** -10)
    pairs, mul = rope_pairs([d], "none", 1.0, 10000.0, 1.0)
    q, k, v = (b["qkv"][:, i * h:(i + 1) * h].view(t, heads, d) for i in range(3))
    assert near(b["q"], rope64(q, pos, pairs, mul, True, False).transpose(0, 1), 2.0 ** -10)
    assert near(b["k"], rope64(k, pos, pairs, mul, True, False).transpose(0, 1), 2.0 ** -10)
    p = torch.softmax(b["q"].double() @ b["k"].double().transpose(1, 2) * d ** -0.5, -1)
    assert near(b["att"].view(t, heads, d).transpose(0, 1), p @ b["v"].double(), 2.0 ** -8)
    x = stream0.double() + gate.double() * step64(b["a8"], b["a8s"], "out")
    assert near(b["x"], x, 2.0 ** -16)
    n2, _ = norm64(b["x"].double(), 2, None, None, 1e-6)
    assert near(b["n2"].double() * wide(b["n2s"], 1, t, h), n2, 2.0 ** -4)
    assert near(b["up"].double() * wide(b["ups"], 1, t, ff), act64(step64(b["n2"], b["n2s"], "up"), "gelu_tanh"), 2.0 ** -4)
    proj = step64(b["up"], b["ups"], "down")
    assert near(b["proj"], proj, 2.0 ** -10)
    y, _ = norm64(b["proj"].double(), 2, None, None, 1e-6)
    assert near(b["y"], b["x"].double() + gate.double() * y, 2.0 ** -16)
    # recorded and replayed on inputs that changed in place
    with torch.cuda.stream(side):
        graph = edb.Graph(round_)
        stream0.mul_(0.5)
        graph.launch()
        replayed = {name: v.clone() for name, v in b.items()}
        round_()
    side.synchronize()
    for name, v in b.items():
        same = bits(v) == bits(replayed[name]) if v.dtype == F8 else v == replayed[name]
        assert bool(same.all()), name
