"""The 8-bit dense layer at the calls between its main ones: transforms and derivatives,
a single row of any stride, non-finite and empty groups through each join of the gated
product, strided operands there, overlapping streams, offsets beyond 32 bits. Bounds as
in test_8bit_dense_layer.py."""

import contextlib
import re
import warnings
from pathlib import Path

import pytest
import torch

from libstrix_b200 import _lib, dense, torch_ops
from oracle import dense as O
from test_8bit_dense_layer import DEV, F8, GATE_REL, check_rows, gemm_case, gemm_error, norm_case, status_ok


# ------------------------------------------------- transforms and derivatives
def calls(device):
    """Each public call on small operands, with the operand that may be wrapped first."""
    x, r, w = (t.to(device) for t in norm_case(4, 256, torch.bfloat16, 1))
    a, sa, wq, sw = (t.to(device) for t in gemm_case(4, 256, 256))
    bias = torch.ones(256, device=device).bfloat16()
    return {
        "norm": (lambda t: dense.rms_norm_quant(t, w, residual=r)[1], x),
        "norm_weight": (lambda t: dense.rms_norm_quant(x, t)[1], w),
        "norm_residual": (lambda t: dense.rms_norm_quant(x, w, residual=t)[1], r),
        "act": (lambda t: dense.act_mul_quant(t)[1], x),
        "gemm_scale": (lambda t: dense.fp8_gemm(a, t, wq, sw), sa),
        "gemm_weight_scale": (lambda t: dense.fp8_gemm(a, sa, wq, t), sw),
        "gemm_bias": (lambda t: dense.fp8_gemm(a, sa, wq, sw, t), bias),
        "gated_scale": (lambda t: dense.fp8_gemm_act_mul_quant(a, t, wq, sw)[1], sa),
    }


class Wrapped(torch.Tensor):
    pass


def test_only_ordinary_calls_skip_the_dispatcher():
    x, w = torch.randn(3, 4), torch.randn(4)
    assert dense._plain(x, w, None)
    assert dense._plain(x, torch.nn.Parameter(w, requires_grad=False))
    assert not dense._plain(x, w.as_subclass(Wrapped)) and not dense._plain(x.as_subclass(Wrapped), w)
    p = torch.nn.Parameter(w)
    assert not dense._plain(x, p)
    with torch.no_grad():
        assert dense._plain(x, p)
    seen = []

    def look(t):
        seen.append(dense._plain(t, w))
        return (t * 2).sum()

    torch.func.vmap(look)(x)
    torch.func.grad(look)(w)
    torch.func.vmap(lambda t: look(x) + t.sum())(x)      # an operand from outside the transform
    assert seen == [False, False, False]


def test_direct_path_needs_no_private_names(monkeypatch):
    monkeypatch.setattr(dense, "_are_functorch_transforms_active", None)
    assert not dense._plain(torch.randn(3))


def test_launches_need_no_private_names(monkeypatch):
    """Without torch's raw device and stream getters _launch uses the public objects."""
    from types import SimpleNamespace

    seen = []
    monkeypatch.setattr(torch_ops, "_raw_stream", None)
    monkeypatch.setattr(torch_ops._lib, "call", lambda *a: seen.append(a))
    monkeypatch.setattr(torch.cuda, "device", lambda dev: contextlib.nullcontext(seen.append(dev)))
    monkeypatch.setattr(torch.cuda, "current_stream", lambda dev: SimpleNamespace(cuda_stream=77))
    torch_ops._launch(SimpleNamespace(get_device=lambda: 3), "strix_entry", 1, 2)
    assert seen == [3, ("strix_entry", 1, 2, 77)]


@pytest.mark.parametrize("name", calls("cpu"))
def test_forward_mode_is_refused(name):
    from torch.autograd import forward_ad

    f, t = calls("cpu")[name]
    with forward_ad.dual_level():
        with pytest.raises(RuntimeError, match="forward-mode"):
            f(forward_ad.make_dual(t, torch.ones_like(t)))
    with pytest.raises(RuntimeError, match="forward-mode"):
        torch.func.jvp(f, (t,), (torch.ones_like(t),))


@pytest.mark.gpu
def test_vmap_runs_the_products_and_names_what_it_cannot():
    x = norm_case(6, 256, torch.bfloat16, 1, False)[0].to(DEV).view(2, 3, 256)
    a, sa, w, sw = (t.to(DEV) for t in gemm_case(6, 256, 256))
    a3, sa3 = a.view(2, 3, 256), sa.view(2, 3, 2)
    with warnings.catch_warnings():
        warnings.simplefilter("ignore")                  # "performance drop": torch's fallback loops
        out = torch.func.vmap(lambda s: dense.fp8_gemm(a3[0], s, w, sw))(sa3)
        s = torch.func.vmap(lambda t: dense.act_mul_quant(t)[1])(x)
    for i in range(2):
        assert torch.equal(out[i], dense.fp8_gemm(a3[0], sa3[i], w, sw))
        assert torch.equal(s[i], dense.act_mul_quant(x[i])[1])
    with pytest.raises(RuntimeError, match="[Bb]atching rule"):
        torch.func.vmap(lambda t: dense.rms_norm_quant(t, w.new_ones(256).bfloat16())[1])(x)


@pytest.mark.gpu
@pytest.mark.parametrize("name", calls("cpu"))
def test_gradients_are_never_lost_silently(name):
    """As through torch.ops.strix: the result carries a node, whose backward pass warns."""
    f, t = calls(DEV)[name]
    want = f(t)
    got = f(t.clone().requires_grad_())
    assert torch.equal(got.detach(), want) and got.grad_fn is not None
    with torch.no_grad():
        assert not f(t.clone().requires_grad_()).requires_grad


# ------------------------------------------------------------------ int8 MLP
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_mlp_blocks_return_the_type_of_their_rows(dtype):
    from torch._subclasses.fake_tensor import FakeTensorMode

    def t(*shape, dtype):
        return torch.empty(*shape, dtype=dtype, device="cuda")

    f32, i8 = torch.float32, torch.int8
    with FakeTensorMode():
        x, w = t(3, 256, dtype=dtype), t(256, dtype=dtype)
        out8 = dense.fused_mlp_int8_w8a8(x, w, t(768, 256, dtype=i8), t(768, dtype=f32), t(256, 384, dtype=i8),
                                         t(256, dtype=f32))
        outf = dense.fused_mlp_fp8_w8a8(x, w, t(768, 256, dtype=F8), t(6, 2, dtype=f32), t(256, 384, dtype=F8),
                                        t(2, 3, dtype=f32))
    assert out8.dtype == dtype and outf.dtype == dtype and out8.shape == outf.shape == (3, 256)


@pytest.mark.gpu
def test_int8_mlp_blocks_chain_in_fp16():
    """The increment of one block is the next block's x, beside the residual stream."""
    t, h, i = 19, 256, 384
    x, r, w = norm_case(t, h, torch.float16, 3)
    g = torch.Generator().manual_seed(4)
    w13 = torch.randint(-127, 128, (2 * i, h), generator=g, dtype=torch.int8).to(DEV)
    w2 = torch.randint(-127, 128, (h, i), generator=g, dtype=torch.int8).to(DEV)
    s13, s2 = (torch.rand(2 * i, generator=g) * 1e-4 + 1e-4).to(DEV), (torch.rand(h, generator=g) * 1e-4).to(DEV)
    xd, rd, wd = x.to(DEV), r.to(DEV), w.to(DEV)
    y = dense.fused_mlp_int8_w8a8(xd, wd, w13, s13, w2, s2, residual=rd, residual_out=rd)
    q, s = dense.rms_norm_quant(xd, wd, residual=r.to(DEV), q_dtype=torch.int8)
    q, s = dense.act_mul_quant(torch.ops.strix.w8a8_int8_gemm(q, s, w13, s13), q_dtype=torch.int8)
    assert torch.equal(y, torch.ops.strix.w8a8_int8_gemm(q, s, w2, s2).half())
    dense.fused_mlp_int8_w8a8(y, wd, w13, s13, w2, s2, residual=rd, residual_out=rd)
    want = ((x.float() + r.float()).half().float() + y.float().cpu()).half()
    assert torch.equal(rd.cpu(), want)


# ---------------------------------------------------------------- vLLM linear
@pytest.mark.parametrize("rows", [0, 3, 9])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_vllm_linear_hands_the_kernels_a_bias_of_their_type(monkeypatch, rows, dtype):
    """With products that refuse what the kernels refuse, and add the bias as they do."""
    from libstrix_b200 import moe
    from strix_vllm import fp8

    def product(q, s, w, scales, bias, out_dtype):
        assert bias is None or bias.dtype == out_dtype and bias.is_contiguous()
        out = torch.zeros(q.size(0), w.size(0)) if bias is None else bias.float().expand(q.size(0), -1)
        return out.to(out_dtype)

    def few(x, w, scales, bias):
        assert 1 <= x.size(0) <= 8 and (bias is None or bias.dtype == torch.bfloat16)
        return product(x, None, w, scales, bias, torch.bfloat16)

    monkeypatch.setattr(moe, "act_quant_fp8", lambda x: (x, None))
    monkeypatch.setattr(dense, "fp8_gemm", product)
    monkeypatch.setattr(fp8, "apply_fp8", few)
    bias = torch.randn(64)[::2].to(dtype)
    out = fp8.apply_fp8_w8a8(torch.zeros(rows, 128).bfloat16(), torch.zeros(32, 128), torch.zeros(1, 1), bias)
    assert out.dtype == torch.bfloat16 and torch.equal(out, bias.bfloat16().expand(rows, -1))


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [0, 3, 9, 100])
def test_vllm_linear_with_an_fp32_bias(rows):
    from strix_vllm import fp8

    x = norm_case(rows, 640, torch.bfloat16, 30, False)[0].to(DEV)
    w, sw = (t.to(DEV) for t in gemm_case(1, 384, 640, 31)[2:])
    bias = torch.randn(384, generator=torch.Generator().manual_seed(5)).to(DEV)
    out, bare = fp8.apply_fp8_w8a8(x, w, sw, bias), fp8.apply_fp8_w8a8(x, w, sw, None)
    status_ok()
    want = bare.double() + bias.double()
    # half a step of the 16-bit sums, and half a step of the result
    assert ((out.double() - want).abs() <= 2.0 ** -8 * (1 + 2.0 ** -8) * (bare.double().abs() + want.abs())).all()


# ------------------------------------------------------- strides of one element
def odd_row(t):
    """The row t [1, K] with a row stride that no kernel could walk."""
    return t.as_strided(t.shape, (t.size(1) + 3, 1))


@pytest.mark.gpu
@pytest.mark.parametrize("q_dtype", [F8, torch.int8])
def test_a_single_row_may_have_any_stride(q_dtype):
    x, r, w = (t.to(DEV) for t in norm_case(1, 256, torch.bfloat16, 6))
    wide = torch.zeros(1, 261, dtype=x.dtype, device=DEV)        # a slice of a matrix of odd width
    wide[:, :256] = x
    want = dense.rms_norm_quant(x, w, residual=r, q_dtype=q_dtype)
    for xx, rr in ((odd_row(x), r), (x, odd_row(r)), (wide[:, :256], odd_row(r)), (x.as_strided((1, 256), (1, 1)), r)):
        out = odd_row(torch.empty_like(r))
        got = dense.rms_norm_quant(xx, w, residual=rr, residual_out=out, q_dtype=q_dtype)
        assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(got, want))
        assert torch.equal(out, (x.float() + r.float()).bfloat16())
    in_place = x.clone()                                         # x itself, under two strides
    dense.rms_norm_quant(in_place, w, residual=r, residual_out=odd_row(in_place), q_dtype=q_dtype)
    assert torch.equal(in_place, (x.float() + r.float()).bfloat16())
    with pytest.raises(RuntimeError, match="apart"):             # half of it stays refused
        both = torch.zeros(1, 512, dtype=x.dtype, device=DEV)
        dense.rms_norm_quant(both[:, :256], w, residual=r, residual_out=both[:, 128:384], q_dtype=q_dtype)
    want = dense.act_mul_quant(x, q_dtype=q_dtype)
    for xx in (odd_row(x), wide[:, :256]):
        got = dense.act_mul_quant(xx, q_dtype=q_dtype)
        assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(got, want))


@pytest.mark.gpu
@pytest.mark.parametrize("n", [256, 144])
def test_a_single_row_of_the_gated_product_may_have_any_stride(n):
    """The C entry, with output strides that only more rows would need."""
    k = 256
    a, sa, w, sw = (t.to(DEV) for t in gemm_case(1, 2 * n, k, 7))
    q, s = dense.fp8_gemm_act_mul_quant(a, sa, w, sw)
    q2, s2 = torch.empty_like(q), torch.empty_like(s)
    ws = torch.empty(2 * n * 4, dtype=torch.uint8, device=DEV)
    torch_ops._launch(a, "strix_w8a8_fp8_gated", q2.data_ptr(), s2.data_ptr(), a.data_ptr(), sa.data_ptr(), w.data_ptr(),
                      sw.data_ptr(), ws.data_ptr(), ws.numel(), 1, n, k, 7, k, 5, 0, *sa.stride(), *sw.stride(), 1)
    status_ok()
    assert torch.equal(q.view(torch.uint8), q2.view(torch.uint8)) and torch.equal(s, s2)


@pytest.mark.gpu
def test_a_bias_of_one_element_may_have_any_stride():
    a, sa, w, sw = (t.to(DEV) for t in gemm_case(5, 1, 256, 8))
    bias = torch.randn(6, device=DEV).bfloat16()
    assert torch.equal(dense.fp8_gemm(a, sa, w, sw, bias[::6]), dense.fp8_gemm(a, sa, w, sw, bias[:1].clone()))


# ------------------------------------------------------ slices of one wider matrix
@pytest.mark.gpu
@pytest.mark.parametrize("q_dtype", [F8, torch.int8])
def test_norm_with_rows_side_by_side_in_one_matrix(q_dtype):
    m, k = 9, 256
    x, r, w = (t.to(DEV) for t in norm_case(m, k, torch.bfloat16, 9))
    want = dense.rms_norm_quant(x, w, residual=r, q_dtype=q_dtype)
    total = (x.float() + r.float()).bfloat16()
    for at_x, at_r, at_out in ((0, 256, 512), (512, 0, 256), (264, 520, 8)):
        wide = torch.full((m, 3 * k + 8), -7.0, dtype=x.dtype, device=DEV)
        wide[:, at_x:at_x + k], wide[:, at_r:at_r + k] = x, r
        out = wide[:, at_out:at_out + k]
        got = dense.rms_norm_quant(wide[:, at_x:at_x + k], w, residual=wide[:, at_r:at_r + k], residual_out=out,
                                   q_dtype=q_dtype)
        assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(got, want))
        assert torch.equal(out, total)
        assert torch.equal(wide[:, at_x:at_x + k], x) and torch.equal(wide[:, at_r:at_r + k], r)
        assert ((wide == -7.0).sum() >= 8 * m).item()


@pytest.mark.gpu
@pytest.mark.parametrize("first", [8, 248, 264, 504, 776, 1016])
def test_norm_refuses_a_sum_that_runs_into_its_input(first):
    """Columns [256, 512) of rows of 768 as input: a sum that starts less than a row's
    width before or behind them, in the same row or the next one."""
    buf = torch.zeros(4 * 768 + 1024, dtype=torch.bfloat16, device=DEV)
    x = buf.as_strided((4, 256), (768, 1), 256)
    out = buf.as_strided((4, 256), (768, 1), first)
    r, w = torch.ones(4, 256, device=DEV).bfloat16(), torch.ones(256, device=DEV).bfloat16()
    with pytest.raises(RuntimeError, match="apart"):
        dense.rms_norm_quant(x, w, residual=r, residual_out=out)
    with pytest.raises(RuntimeError, match="apart"):
        dense.rms_norm_quant(r, w, residual=x, residual_out=out)


# ------------------------------------------------------------- gated product's joins
# One shape per way that the sums reach the gate: the weight stream's join (two tile
# widths), the wide kernel's registers and its join along K, and fp32 rows through the
# workspace (gate and up rows that share a weight block) from either kernel.
JOINS = {
    "stream16": (9, 384, 656),
    "stream32": (20, 384, 4112),
    "wide": (70, 384, 640),
    "wide_split": (70, 256, 6016),
    "rows_stream": (9, 144, 656),
    "rows_wide": (70, 400, 640),
}


def gated_case(join, seed):
    m, n, k = JOINS[join]
    a, sa, w, sw = gemm_case(m, 2 * n, k, seed)
    return m, n, k, a, sa * 0.03, w, sw


def gated(a, sa, w, sw, activation="silu"):
    q, s = dense.fp8_gemm_act_mul_quant(a.to(DEV), sa.to(DEV), w.to(DEV), sw.to(DEV), activation)
    status_ok()
    return q.cpu().view(torch.uint8), s.cpu()


def same_outside(got, want, rows=None, group=None):
    """Equal to the bit except in the given rows, or in one group of 128 columns."""
    keep = torch.ones(want[1].shape, dtype=torch.bool)
    if rows is not None:
        keep[rows] = False
    if group is not None:
        keep[:, group] = False
    wide = O.spread(keep, want[0].size(1), 128)
    return torch.equal(got[1][keep], want[1][keep]) and torch.equal(got[0][wide], want[0][wide])


@pytest.mark.gpu
@pytest.mark.parametrize("activation", ["silu", "gelu_tanh"])
@pytest.mark.parametrize("join", JOINS)
def test_gated_product_shows_nan_and_infinity_where_they_are(join, activation):
    m, n, k, a, sa, w, sw = gated_case(join, 70)
    want = gated(a, sa, w, sw, activation)
    bad = a.clone()
    bad.view(torch.uint8)[1, 300] = 0x7F                 # a NaN in a token: its row, every group
    got = gated(bad, sa, w, sw, activation)
    assert got[1][1].isnan().all() and same_outside(got, want, rows=[1])
    for row, group in ((130, 1), (n + 5, 0)):            # in a gate row, in an up row: its group
        bad = w.clone()
        bad.view(torch.uint8)[row, k - 1] = 0x7F
        got = gated(a, sa, bad, sw, activation)
        assert got[1][:, group].isnan().all() and same_outside(got, want, group=group)
    for value in (float("inf"), -float("inf"), float("nan")):   # in a token's scale
        bad = sa.clone()
        bad[m - 1, 2] = value
        got = gated(a, bad, w, sw, activation)
        assert not got[1][m - 1].isfinite().any() and same_outside(got, want, rows=[m - 1])


@pytest.mark.gpu
@pytest.mark.parametrize("join", JOINS)
def test_gated_product_of_zeros_and_of_groups_of_zeros(join):
    m, n, k, a, sa, w, sw = gated_case(join, 71)
    want = gated(a, sa, w, sw)
    zero = a.clone()
    zero.view(torch.uint8)[[0, m - 1]] = 0               # tokens of zeros
    got = gated(zero, sa, w, sw)
    assert (got[1][[0, m - 1]] == 1).all() and not (got[0][[0, m - 1]] & 0x7F).any()
    assert same_outside(got, want, rows=[0, m - 1])
    for first in (128, n + 128):                         # gate rows, or up rows, of the second group
        last = min(first + 128, n if first < n else 2 * n)
        zero = w.clone()
        zero.view(torch.uint8)[first:last] = 0
        got = gated(a, sa, zero, sw)
        assert (got[1][:, 1] == 1).all() and not (got[0][:, 128:256] & 0x7F).any()
        assert same_outside(got, want, group=1)


@pytest.mark.gpu
@pytest.mark.parametrize("join", JOINS)
def test_gated_product_of_strided_operands(join):
    """Rows inside wider matrices, scales stored column-major and inside wider ones."""
    m, n, k, a, sa, w, sw = gated_case(join, 72)
    want = gated(a, sa, w, sw)
    # NaN bytes around the operands must not be read into the result
    wa = torch.full((m, k + 112), 0x7F, dtype=torch.uint8, device=DEV)
    ww = torch.full((2 * n, k + 48), 0x7F, dtype=torch.uint8, device=DEV)
    wa[:, 16:16 + k], ww[:, 32:32 + k] = a.view(torch.uint8).to(DEV), w.view(torch.uint8).to(DEV)
    sws = torch.full((2 * sw.size(0), 3 * sw.size(1)), float("nan"), device=DEV)
    sws[::2, ::3] = sw.to(DEV)
    got = gated(wa.view(F8)[:, 16:16 + k], sa.to(DEV).t().contiguous().t(), ww.view(F8)[:, 32:32 + k], sws[::2, ::3])
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.gpu
def test_gated_products_on_streams_that_overlap():
    """Every join on every stream at once; the workspaces of the fp32 rows are a call's own."""
    cases = [[t.to(DEV) for t in gated_case(join, 73)[3:]] for join in JOINS]
    want = [dense.fp8_gemm_act_mul_quant(*c) for c in cases]
    streams = [torch.cuda.Stream() for _ in range(4)]
    torch.cuda.synchronize()
    got = []
    for i in range(4 * len(cases)):
        with torch.cuda.stream(streams[i % 4]):
            at = (i + i // 4) % len(cases)
            got.append((at, dense.fp8_gemm_act_mul_quant(*cases[at])))
    torch.cuda.synchronize()
    status_ok()
    for at, (q, s) in got:
        assert torch.equal(q.view(torch.uint8), want[at][0].view(torch.uint8)) and torch.equal(s, want[at][1])


@pytest.mark.gpu
@pytest.mark.parametrize("n", [32768, 32784])
def test_gated_product_beyond_32_bit_offsets(n):
    """2.3 billion outputs, and for the second width as many pairs of fp32 rows: the rows at
    both ends against the oracle, the zeros between."""
    m, k = 70000, 144
    a, sa, w, sw = gemm_case(64, 2 * n, k, 74)
    sa = sa * 0.03
    big_a = torch.zeros(m, k, device=DEV).to(F8)
    big_sa = torch.ones(m, 2, device=DEV)
    at = torch.cat([torch.arange(0, 32), torch.arange(m - 32, m)])
    big_a.view(torch.uint8)[at.to(DEV)] = a.view(torch.uint8).to(DEV)
    big_sa[at.to(DEV)] = sa.to(DEV)
    q, s = dense.fp8_gemm_act_mul_quant(big_a, big_sa, w.to(DEV), sw.to(DEV))
    status_ok()
    h, e = O.fp8_gemm(a, sa, w, sw), gemm_error(a, sa, w, sw)
    err = 1.13 * e[:, :n] * (h[:, n:].abs() + e[:, n:]) + h[:, :n].abs() * e[:, n:]
    check_rows(q[at.to(DEV)], s[at.to(DEV)], O.act_mul(h, "silu"), True, GATE_REL, err)
    assert (s[32:m - 32] == 1).all()
    for lo in range(32, m - 32, 9000):                   # a piece at a time: no second copy of it all
        assert not (q[lo:min(lo + 9000, m - 32)].view(torch.uint8) & 0x7F).any()


# -------------------------------------------------------------------- the build
def test_kernel_sources_have_no_switches():
    """What the kernels do is chosen by sizes, types and alignment at run time: no part of a
    source is compiled in or out."""
    csrc = Path(dense.__file__).parent / "csrc"
    found = [f"{f.name}:{i}" for f in sorted(csrc.iterdir()) for i, line in enumerate(f.read_text().splitlines(), 1)
             if re.match(r"\s*#\s*(if|ifdef|ifndef|elif)\b", line)]
    assert not found


def test_gated_workspace_of_sizes_beyond_63_bits():
    size = _lib.load().strix_w8a8_fp8_gated_workspace
    m, n = (1 << 31) - 257, (1 << 30) - 144
    assert m * 8 * n > 2 ** 63 and size(m, n, 16) == -1
    assert size(m, (1 << 30) - 256, 16) == 0              # one kernel: no rows in between
    m = 2 ** 63 // (8 * n)                                # the most that 63 bits hold
    assert size(m, n, 16) == m * 8 * n and size(m + 1, n, 16) == -1
    assert size(70000, 144, 16) == 70000 * 144 * 8


@pytest.mark.gpu
def test_first_calls_from_many_threads():
    """A C call gives up the interpreter's lock, so the first calls of a process may meet in
    the tables that they fill."""
    import subprocess
    import sys

    code = """
import threading, torch
from libstrix_b200 import dense
f8 = torch.float8_e4m3fn
torch.manual_seed(0)
x = torch.randn(300, 2048, device="cuda").bfloat16()
nw = torch.ones(2048, device="cuda").bfloat16()
w13, w2 = torch.randn(1024, 2048, device="cuda").to(f8), torch.randn(2048, 512, device="cuda").to(f8)
s13, s2 = torch.rand(8, 16, device="cuda"), torch.rand(16, 4, device="cuda")
rows = (3, 20, 50, 300)
out, gate = [None] * 16, threading.Barrier(16)
torch.cuda.synchronize()

def work(i):
    stream = torch.cuda.Stream()
    gate.wait()
    with torch.cuda.stream(stream):
        out[i] = dense.fused_mlp_fp8_w8a8(x[:rows[i % 4]], nw, w13, s13, w2, s2)
    stream.synchronize()

threads = [threading.Thread(target=work, args=(i,)) for i in range(16)]
[t.start() for t in threads]
[t.join() for t in threads]
for i in range(16):
    assert torch.equal(out[i], dense.fused_mlp_fp8_w8a8(x[:rows[i % 4]], nw, w13, s13, w2, s2)), i
"""
    subprocess.run([sys.executable, "-c", code], check=True, timeout=240, cwd=Path(__file__).resolve().parent.parent)


# ------------------------------------------------- ends of the fp32 arithmetic
@pytest.mark.gpu
@pytest.mark.parametrize("q_dtype", [F8, torch.int8])
def test_norm_of_rows_whose_squares_leave_fp32(q_dtype):
    """As the header says: zeros, and the other rows as they are."""
    x, _, w = (t if t is None else t.to(DEV) for t in norm_case(3, 256, torch.bfloat16, 10, False))
    want = dense.rms_norm_quant(x, w, q_dtype=q_dtype)
    x[1] = 1e25
    q, s = dense.rms_norm_quant(x, w, q_dtype=q_dtype)
    assert not q[1].float().any() and (s[1] == 1).all()
    assert torch.equal(q.view(torch.uint8)[::2], want[0].view(torch.uint8)[::2]) and torch.equal(s[::2], want[1][::2])


@pytest.mark.gpu
@pytest.mark.parametrize("m", [5, 100])
def test_product_of_scales_that_leave_fp32(m):
    """As the header says: the two scales are multiplied first. Below 2^-126 a block adds
    nothing, beyond 2^128 it is not finite; up to those ends it is exact."""
    n, k = 128, 256
    a = torch.ones(m, k, device=DEV).to(F8)
    w = torch.ones(n, k, device=DEV).to(F8)
    sa, sw = torch.ones(m, 2, device=DEV), torch.ones(1, 2, device=DEV)

    def first_block(x, y):
        sa[:, 0], sw[:, 0] = x, y
        return dense.fp8_gemm(a, sa, w, sw, out_dtype=torch.float32)

    assert (first_block(2.0 ** -60, 2.0 ** -70) == 128).all()
    assert not first_block(2.0 ** 70, 2.0 ** 60).isfinite().any()
    sa[:, 1] = 0
    assert (first_block(2.0 ** -60, 2.0 ** -66) == 128 * 2.0 ** -126).all()
    assert (first_block(2.0 ** 60, 2.0 ** 60) == 128 * 2.0 ** 120).all()
