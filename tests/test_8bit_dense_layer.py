"""The 8-bit dense layer against the 64-bit oracle: norm and gated activation into 8
bits, the FP8 product with block scales and its gated form, and the MLP that runs them.

Bounds. u = 2^-24 is half a step of fp32, relative to the value.
  * norm: a thread adds at most 64 squares in a row and the CTA adds the threads' sums in
    two trees of 5 steps, a square itself is rounded, so the mean is off by at most 76 u;
    the root halves that; root, mean, three products: fewer than 10 u more. y is within
    48 u + a margin = 2^-18 of the formula, and so is a scale.
  * gate: __expf(x) is documented to 2 + 1.173 |x| steps of 2^-23; the gelu's argument
    adds |x| * 5 u. With |x| <= 80 (beyond it both sides are below 1e-33 |up|) that is below
    2^-14 of the value.
  * a product of two e4m3 values is exact in fp32 (8 bits). Each of the 128 additions
    of a K block is given a whole step of fp32 (2 u: tensor cores may truncate), each
    of the fold's products and additions u: |error| <= u (256 + 3 + blocks) * sum of
    |terms|, and half a step of the output's type.
  * an 8-bit value is within half a step of the quotient, and what moved the quotient.
"""

import ctypes

import pytest
import torch

import libstrix_b200 as strix
from libstrix_b200 import _lib, dense
from oracle import dense as O

DEV = "cuda"
F8 = torch.float8_e4m3fn
U = 2.0 ** -24
Y_REL = 2.0 ** -18
GATE_REL = 2.0 ** -14
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: U}


def gen(seed):
    return torch.Generator().manual_seed(seed)


def status_ok():
    flag = ctypes.c_int32(-1)
    assert _lib.load().strix_umma_status(ctypes.byref(flag)) == 0 and flag.value == 0


def half_step_e4m3(v):
    _, e = torch.frexp(v)
    return torch.ldexp(torch.ones_like(v), e.clamp_min(-5) - 5)


def check_rows(q, s, y, fp8, rel, err=None):
    """q, s (of the kernel) against 64-bit rows y that it may know to `rel` of the value,
    and to `err` absolutely (a tensor like y)."""
    v, s_ref = O.quantise(y, fp8)
    s, q = s.double().cpu(), q.cpu()
    err = torch.zeros_like(y) if err is None else err
    err = err + rel * y.abs()
    if fp8:
        worst = O.group_scales(err, 448.0, 128) * (err.abs().amax() > 0)
        full, wide = O.spread(s_ref, y.size(1), 128), O.spread(worst, y.size(1), 128)
    else:
        worst = err.amax(-1) / 127
        full, wide = s_ref[:, None], worst[:, None]
    one = (s_ref == 1)   # all-zero groups
    assert ((s - s_ref).abs() <= torch.where(one, 0.0, worst + 4 * U * s_ref)).all(), "scales"
    moved = err / full + v.abs() * (wide / full + 8 * U)
    step = half_step_e4m3(v) if fp8 else torch.full_like(v, 0.5)
    off = (q.double() - v).abs()
    assert (off <= step + moved).all(), ("8-bit values", (off - step - moved).max().item())


# ------------------------------------------------------------------------- norm
def norm_case(m, k, dtype, seed, residual=True, w_dtype=None):
    g = gen(seed)
    x = (torch.randn(m, k, generator=g) * torch.exp(torch.randn(m, 1, generator=g))).to(dtype)
    r = (torch.randn(m, k, generator=g) * 3).to(dtype) if residual else None
    w = (1 + 0.3 * torch.randn(k, generator=g)).to(w_dtype or dtype)
    return x, r, w


def check_norm(x, r, w, eps, q_dtype, out=None):
    xd, rd, wd = x.to(DEV), None if r is None else r.to(DEV), w.to(DEV)
    ro = None if r is None else torch.empty_like(rd)
    q, s = dense.rms_norm_quant(xd, wd, eps, rd, ro, q_dtype=q_dtype)
    torch.cuda.synchronize()
    total, y = O.rms_norm(x, w, eps, r)
    check_rows(q, s, y, q_dtype == F8, Y_REL)
    if r is not None:
        assert torch.equal(ro.cpu(), (x.float() + r.float()).to(x.dtype))
    assert torch.equal(xd.cpu(), x)
    return q, s


@pytest.mark.gpu
@pytest.mark.parametrize("q_dtype", [F8, torch.int8])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m,k", [(1, 16), (3, 64), (2, 128), (5, 144), (7, 2048), (33, 2880), (9, 5120),
                                 (2, 8192), (3, 8208), (2, 16384), (2, 17408), (1, 32784), (1, 65536)])
def test_norm(m, k, dtype, q_dtype):
    for residual in (True, False):
        x, r, w = norm_case(m, k, dtype, m * 7 + k, residual)
        check_norm(x, r, w, 1e-6, q_dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_norm_with_fp32_weight_and_large_eps(dtype):
    x, r, w = norm_case(6, 1040, dtype, 3, True, torch.float32)
    for q_dtype in (F8, torch.int8):
        check_norm(x, r, w, 0.5, q_dtype)


@pytest.mark.gpu
def test_norm_int8_takes_widths_off_16():
    for m, k in ((4, 1000), (3, 8), (400, 24)):
        x, r, w = norm_case(m, k, torch.bfloat16, 4)
        check_norm(x, r, w, 1e-5, torch.int8)


@pytest.mark.gpu
def test_norm_many_rows():
    x, r, w = norm_case(4097, 512, torch.bfloat16, 5)
    check_norm(x, r, w, 1e-6, F8)


@pytest.mark.gpu
@pytest.mark.parametrize("q_dtype", [F8, torch.int8])
def test_norm_updates_the_residual_in_place(q_dtype):
    x, r, w = norm_case(17, 2880, torch.bfloat16, 6)
    xd, rd, wd = x.to(DEV), r.to(DEV), w.to(DEV)
    want = dense.rms_norm_quant(xd, wd, 1e-6, rd, None, q_dtype=q_dtype)
    assert torch.equal(rd.cpu(), r)                      # not stored: left alone
    for target in ("residual", "x"):
        a, b = xd.clone(), rd.clone()
        t = b if target == "residual" else a
        got = dense.rms_norm_quant(a, wd, 1e-6, b, t, q_dtype=q_dtype)
        assert torch.equal(t.cpu(), (x.float() + r.float()).to(x.dtype))
        assert torch.equal((a if t is b else b).cpu(), x if t is b else r)
        for u, v in zip(got, want):
            assert torch.equal(u.view(torch.uint8), v.view(torch.uint8))


@pytest.mark.gpu
def test_norm_reads_strided_rows():
    """x and the residual as column slices of wider matrices, the sum into a third."""
    x, r, w = norm_case(11, 640, torch.bfloat16, 7)
    wide = torch.full((11, 1024), float("nan"), dtype=x.dtype, device=DEV)
    wide_r, wide_o = wide.clone(), wide.clone()
    wide[:, 64:704], wide_r[:, 128:768] = x.to(DEV), r.to(DEV)
    q, s = dense.rms_norm_quant(wide[:, 64:704], w.to(DEV), 1e-6, wide_r[:, 128:768], wide_o[:, 8:648])
    _, y = O.rms_norm(x, w, 1e-6, r)
    check_rows(q, s, y, True, Y_REL)
    assert torch.equal(wide_o[:, 8:648].cpu(), (x.float() + r.float()).to(x.dtype))
    assert wide_o[:, :8].isnan().all() and wide_o[:, 648:].isnan().all()
    # one row for all: a broadcast input
    q1, s1 = dense.rms_norm_quant(x[:1].to(DEV).expand(11, 640), w.to(DEV))
    assert torch.equal(q1.view(torch.uint8), q1[:1].expand(11, 640).contiguous().view(torch.uint8))
    check_rows(q1[:1], s1[:1], O.rms_norm(x[:1], w, 1e-6)[1], True, Y_REL)


@pytest.mark.gpu
@pytest.mark.parametrize("q_dtype", [F8, torch.int8])
def test_norm_of_zeros_and_of_groups_of_zeros(q_dtype):
    x, r, w = norm_case(4, 512, torch.bfloat16, 8)
    x[1], r[1] = 0, 0
    x[2, 128:256], r[2, 128:256] = 0, 0
    w[384:] = 0
    q, s = check_norm(x, r, w, 1e-6, q_dtype)
    assert not q[1].float().any() and (s[1] == 1).all()
    if q_dtype == F8:
        assert s[2, 1] == 1 and (s[:, 3] == 1).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_norm_of_tiny_and_huge_values(dtype):
    """Values next to the ends of the type: sums of squares that stay inside fp32."""
    big = 60000.0 if dtype == torch.float16 else 1e17
    small = 6e-5 if dtype == torch.float16 else 1e-17
    x, _, w = norm_case(2, 256, dtype, 9, False)
    x = x.sign() * (x.float().abs() % 1 + 0.5)
    for scale in (big / 2, small):
        check_norm((x * scale).to(dtype), None, w, 0.0, F8)


@pytest.mark.gpu
@pytest.mark.parametrize("q_dtype", [F8, torch.int8])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_norm_shows_nan_and_infinity_in_its_own_row_only(bad, q_dtype):
    x, r, w = norm_case(5, 384, torch.bfloat16, 10)
    clean = dense.rms_norm_quant(x.to(DEV), w.to(DEV), 1e-6, r.to(DEV), q_dtype=q_dtype)
    y = x.clone()
    y[2, 200] = bad
    q, s = dense.rms_norm_quant(y.to(DEV), w.to(DEV), 1e-6, r.to(DEV), q_dtype=q_dtype)
    rows = [0, 1, 3, 4]
    assert torch.equal(q.view(torch.uint8)[rows], clean[0].view(torch.uint8)[rows])
    assert torch.equal(s[rows], clean[1][rows])
    assert not s[2].isfinite().all()                     # the row's damage is seen


# ------------------------------------------------------------- gated activation
@pytest.mark.gpu
@pytest.mark.parametrize("activation", ["silu", "gelu_tanh"])
@pytest.mark.parametrize("q_dtype", [F8, torch.int8])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("m,k", [(1, 16), (2, 128), (3, 144), (5, 768), (33, 2880), (2, 17408), (1, 33008)])
def test_act_mul(m, k, dtype, q_dtype, activation):
    x = (torch.randn(m, 2 * k, generator=gen(m + k)) * 4).to(dtype)
    q, s = dense.act_mul_quant(x.to(DEV), activation, q_dtype=q_dtype)
    assert q.shape == (m, k) and q.dtype == q_dtype
    check_rows(q, s, O.act_mul(x, activation), q_dtype == F8, GATE_REL)


@pytest.mark.gpu
@pytest.mark.parametrize("activation", ["silu", "gelu_tanh"])
def test_act_mul_ends_of_the_gate(activation):
    """Strongly negative gates give 0, strongly positive ones the gate itself."""
    g = torch.tensor([-1e4, -200.0, -100.0, -88.0, -30.0, -1.0, -0.0, 0.0, 1.0, 30.0, 88.0, 100.0, 200.0, 1e4, 5.0, -5.0])
    x = torch.cat([g, torch.ones(16)])[None].to(DEV)
    q, s = dense.act_mul_quant(x, activation)
    y = O.act_mul(x.cpu(), activation)
    assert q.float().isfinite().all()
    check_rows(q, s, y, True, GATE_REL, torch.full_like(y, 1e-30))


@pytest.mark.gpu
def test_act_mul_strided_many_rows_zeros_and_nan():
    m, k = 1000, 272
    x = torch.randn(m, 2 * k, generator=gen(1)).bfloat16()
    x[5] = 0
    x[6, 128:256] = 0
    wide = torch.full((m, 2 * k + 24), float("nan"), dtype=x.dtype, device=DEV)
    wide[:, 16:16 + 2 * k] = x.to(DEV)
    y = O.act_mul(x, "silu")
    for q_dtype in (F8, torch.int8):
        q, s = dense.act_mul_quant(wide[:, 16:16 + 2 * k], "silu", q_dtype=q_dtype)
        check_rows(q, s, y, q_dtype == F8, GATE_REL)
        bad = x.clone()
        bad[9, 3] = float("nan")
        bad[11, k + 200] = float("inf")
        q2, s2 = dense.act_mul_quant(bad.to(DEV), "silu", q_dtype=q_dtype)
        assert s2.reshape(m, -1)[9].isnan().any() and not s2.reshape(m, -1)[11].isfinite().all()
        rows = [i for i in range(m) if i not in (9, 11)]
        assert torch.equal(s2[rows], s[rows]) and torch.equal(q2.view(torch.uint8)[rows], q.view(torch.uint8)[rows])
        if q_dtype == F8:
            assert s2[9].isnan().sum() == 1              # only the group that holds it


# ------------------------------------------------------------------ FP8 product
def gemm_case(m, n, k, seed=0):
    g = gen(seed * 7919 + m * 31 + n * 17 + k)
    a = (torch.randn(m, k, generator=g) * 60).clamp(-448, 448).to(F8)
    w = (torch.randn(n, k, generator=g) * 60).clamp(-448, 448).to(F8)
    kb, nb = (k + 127) // 128, (n + 127) // 128
    sa = torch.rand(m, kb, generator=g) * 4e-2 + 1e-3
    sw = torch.rand(nb, kb, generator=g) * 9e-3 + 1e-4
    return a, sa, w, sw


def gemm_error(a, sa, w, sw):
    """The bound on the fp32 sums, without the output's rounding."""
    blocks = sa.size(1)
    return U * (256 + 3 + blocks) * O.fp8_gemm(a.float().abs(), sa, w.float().abs(), sw)


def check_gemm(m, n, k, seed=0, out_dtype=torch.bfloat16, bias=False):
    a, sa, w, sw = gemm_case(m, n, k, seed)
    b = torch.randn(n, generator=gen(seed)).to(out_dtype) if bias else None
    out = dense.fp8_gemm(a.to(DEV), sa.to(DEV), w.to(DEV), sw.to(DEV), None if b is None else b.to(DEV), out_dtype)
    status_ok()
    assert out.dtype == out_dtype and tuple(out.shape) == (m, n)
    ref = O.fp8_gemm(a, sa, w, sw, b)
    err = gemm_error(a, sa, w, sw) + U * ref.abs()
    bound = err + HALF[out_dtype] * (ref.abs() + err) + (2.0 ** -25 if out_dtype == torch.float16 else 0)
    off = (out.double().cpu() - ref).abs()
    assert (off <= bound).all(), ((off - bound).max().item(), off.max().item())


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 2, 15, 16, 17, 32, 33, 64, 65, 100, 128, 129, 256, 257, 300])
@pytest.mark.parametrize("n,k", [(2048, 2048), (1024, 768), (256, 4096)])
def test_gemm(m, n, k):
    check_gemm(m, n, k)


@pytest.mark.gpu
@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("m,n,k", [(1, 1, 16), (1, 8, 128), (3, 127, 144), (16, 129, 272), (20, 200, 112),
                                   (64, 1000, 400), (100, 257, 128), (129, 2055, 256), (257, 520, 1168),
                                   (1000, 777, 528), (300, 5760, 2880)])
def test_gemm_ragged(m, n, k, out_dtype):
    check_gemm(m, n, k, seed=1, out_dtype=out_dtype, bias=True)


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", [(1, 34816, 5120), (16, 5120, 17408), (700, 2560, 5120), (1500, 1024, 2048),
                                   (128, 5120, 17408), (100, 1000, 8192), (65, 513, 16384), (250, 4000, 5120)])
def test_gemm_at_layer_widths(m, n, k):
    check_gemm(m, n, k, seed=2)


@pytest.mark.gpu
@pytest.mark.parametrize("kind,dtype", [(0, torch.bfloat16), (1, torch.float16), (2, torch.float32)])
@pytest.mark.parametrize("m,n", [(1, 77), (40, 77), (70, 333), (300, 701)])
def test_gemm_into_rows_of_a_wider_matrix(m, n, kind, dtype):
    """The C entry with an output stride: rows on 16-byte boundaries (they leave by TMA in the
    wide kernel) and off them; what lies beside the output stays as it was."""
    k = 400
    a, sa, w, sw = (t.to(DEV) for t in gemm_case(m, n, k, 14))
    want = dense.fp8_gemm(a, sa, w, sw, out_dtype=dtype)
    for width, first in ((n + 64 - n % 64 + 64, 16), (n + 37, 3)):
        wide = torch.full((m + 2, width), -7.0, dtype=dtype, device=DEV)
        out = wide[1:m + 1, first:first + n]
        _lib.call("strix_w8a8_fp8_gemm", out.data_ptr(), a.data_ptr(), sa.data_ptr(), w.data_ptr(), sw.data_ptr(),
                  None, m, n, k, k, k, width, *sa.stride(), *sw.stride(), kind,
                  torch.cuda.current_stream().cuda_stream)
        status_ok()
        assert torch.equal(out, want)
        rest = wide.clone()
        rest[1:m + 1, first:first + n] = -7.0
        assert (rest == -7.0).all()


@pytest.mark.gpu
def test_gated_product_into_rows_of_a_wider_matrix():
    for m in (9, 200):
        n, k = 256, 272
        a, sa, w, sw = (t.to(DEV) for t in gemm_case(m, 2 * n, k, 15))
        q, s = dense.fp8_gemm_act_mul_quant(a, sa, w, sw)
        wide = torch.full((m + 2, n + 48), 9.0, device=DEV).to(F8)
        wide_s = torch.full((m + 2, 5), -7.0, device=DEV)
        nbytes = _lib.load().strix_w8a8_fp8_gated_workspace(m, n, k)
        ws = torch.empty(max(nbytes, 16), dtype=torch.uint8, device=DEV)
        out, out_s = wide[1:m + 1, 16:16 + n], wide_s[1:m + 1, 1:3]
        _lib.call("strix_w8a8_fp8_gated", out.data_ptr(), out_s.data_ptr(), a.data_ptr(), sa.data_ptr(), w.data_ptr(),
                  sw.data_ptr(), ws.data_ptr(), nbytes, m, n, k, k, k, n + 48, 5, *sa.stride(), *sw.stride(), 1,
                  torch.cuda.current_stream().cuda_stream)
        status_ok()
        assert torch.equal(out.view(torch.uint8), q.view(torch.uint8)) and torch.equal(out_s, s)
        rest, rest_s = wide.float(), wide_s.clone()
        rest[1:m + 1, 16:16 + n], rest_s[1:m + 1, 1:3] = 9.0, -7.0
        assert (rest == 9.0).all() and (rest_s == -7.0).all()


@pytest.mark.gpu
def test_gemm_long_reduction():
    check_gemm(4, 256, 128 * 1030 + 16, seed=3)
    check_gemm(300, 256, 128 * 1030 + 16, seed=3)


@pytest.mark.gpu
def test_gemm_is_exact_where_every_sum_is():
    """Small whole numbers and scales that are powers of two: each sum fits 24 bits, so
    no order of additions rounds, and the output is the formula's to the bit."""
    for m, n, k in ((7, 300, 640), (200, 520, 1040), (600, 1300, 384)):
        g = gen(k)
        a = torch.randint(-8, 9, (m, k), generator=g).float().to(F8)
        w = torch.randint(-8, 9, (n, k), generator=g).float().to(F8)
        kb = (k + 127) // 128
        sa = torch.pow(2.0, torch.randint(-1, 2, (m, kb), generator=g).float())
        sw = torch.pow(2.0, torch.randint(-1, 2, ((n + 127) // 128, kb), generator=g).float())
        out = dense.fp8_gemm(a.to(DEV), sa.to(DEV), w.to(DEV), sw.to(DEV), out_dtype=torch.float32)
        assert torch.equal(out.cpu().double(), O.fp8_gemm(a, sa, w, sw))


@pytest.mark.gpu
@pytest.mark.parametrize("m", [3, 40, 300])
def test_gemm_strided_operands(m):
    """Rows inside wider matrices, scales stored column-major and inside wider ones."""
    n, k = 392, 656
    a, sa, w, sw = gemm_case(m, n, k, 4)
    want = dense.fp8_gemm(a.to(DEV), sa.to(DEV), w.to(DEV), sw.to(DEV))
    # NaN bytes around the operands must not be read into the result
    wa = torch.full((m, 1024), 0x7F, dtype=torch.uint8, device=DEV).view(F8)
    ww = torch.full((n, 1024), 0x7F, dtype=torch.uint8, device=DEV).view(F8)
    wa.view(torch.uint8)[:, 16:16 + k] = a.view(torch.uint8).to(DEV)
    ww.view(torch.uint8)[:, 32:32 + k] = w.view(torch.uint8).to(DEV)
    sat = sa.to(DEV).t().contiguous().t()
    sww = torch.full((8, 20), float("nan"), device=DEV)
    sww[::2, ::3][:sw.size(0), :sw.size(1)] = sw.to(DEV)
    got = dense.fp8_gemm(wa[:, 16:16 + k], sat, ww[:, 32:32 + k], sww[::2, ::3][:sw.size(0), :sw.size(1)])
    status_ok()
    assert torch.equal(got, want)


@pytest.mark.gpu
@pytest.mark.parametrize("m", [5, 200])
def test_gemm_keeps_nan_and_infinity_in_their_row_or_column(m):
    n, k = 320, 512
    a, sa, w, sw = gemm_case(m, n, k, 5)
    a.view(torch.uint8)[1, 77] = 0x7F
    w.view(torch.uint8)[130, 5] = 0x7F
    sa[3, 2] = float("inf")
    out = dense.fp8_gemm(a.to(DEV), sa.to(DEV), w.to(DEV), sw.to(DEV)).cpu()
    assert out[1].isnan().all() and out[:, 130].isnan().all() and not out[3].isfinite().any()
    rows = [i for i in range(m) if i not in (1, 3)]
    cols = [j for j in range(n) if j != 130]
    assert out[rows][:, cols].isfinite().all()


@pytest.mark.gpu
def test_empty_batches():
    a, sa, w, sw = (t.to(DEV) for t in gemm_case(0, 256, 256))
    assert dense.fp8_gemm(a, sa, w, sw).shape == (0, 256)
    q, s = dense.fp8_gemm_act_mul_quant(a, sa, w, sw)
    assert q.shape == (0, 128) and s.shape == (0, 1)
    x = torch.empty(0, 512, dtype=torch.bfloat16, device=DEV)
    for q_dtype in (F8, torch.int8):
        assert dense.act_mul_quant(x, q_dtype=q_dtype)[0].shape == (0, 256)
        q, s = dense.rms_norm_quant(x, torch.ones(512, dtype=x.dtype, device=DEV), residual=x, residual_out=x,
                                    q_dtype=q_dtype)
        assert q.shape == (0, 512) and s.size(0) == 0


# ----------------------------------------------------------- gated FP8 product
@pytest.mark.gpu
@pytest.mark.parametrize("activation", ["silu", "gelu_tanh"])
@pytest.mark.parametrize("m,n,k", [(1, 16, 128), (2, 768, 2048), (16, 144, 272), (33, 512, 384), (65, 400, 1040),
                                   (256, 768, 2048), (300, 640, 528), (1000, 1024, 2048), (515, 2880, 1152),
                                   (17, 1152, 528), (40, 256, 1040), (64, 768, 2048), (70, 256, 4112), (300, 384, 6016),
                                   (257, 128, 9000 // 16 * 16)])
def test_gated_product(m, n, k, activation):
    a, sa, w, sw = gemm_case(m, 2 * n, k, 6)
    sa = sa * 0.03                                       # gates of a few units
    q, s = dense.fp8_gemm_act_mul_quant(a.to(DEV), sa.to(DEV), w.to(DEV), sw.to(DEV), activation)
    status_ok()
    h, e = O.fp8_gemm(a, sa, w, sw), gemm_error(a, sa, w, sw)
    y = O.act_mul(h, activation)
    # the gates' slopes are at most 1.13; act(g) <= |g|
    err = 1.13 * e[:, :n] * (h[:, n:].abs() + e[:, n:]) + h[:, :n].abs() * e[:, n:]
    check_rows(q, s, y, True, GATE_REL, err)


# ------------------------------------------------------------- used as a layer
def mlp_case(t, h, i, seed=0, dtype=torch.bfloat16):
    g = gen(seed + t + h + i)
    x, r, w = norm_case(t, h, dtype, seed + 1)

    def weights(n, k):
        v = torch.randn(n, k, generator=g) * 0.02
        kb, nb = (k + 127) // 128, (n + 127) // 128
        p = torch.zeros(nb * 128, kb * 128)
        p[:n, :k] = v
        s = p.view(nb, 128, kb, 128).abs().amax((1, 3)) / 448
        full = s.repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)[:, :k]
        return (v / full).to(F8), s

    return (x, w, *weights(2 * i, h), *weights(h, i), r)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("t,h,i", [(1, 512, 768), (40, 2880, 1152), (300, 1024, 1408)])
def test_mlp_fp8_is_its_steps(t, h, i, dtype):
    """The block against its steps, and against a 64-bit MLP of the kernels' own 8-bit rows."""
    x, w, w13, s13, w2, s2, r = mlp_case(t, h, i, dtype=dtype)
    d = [v.to(DEV) for v in (x, w, w13, s13, w2, s2)]
    rd = r.to(DEV)
    out = dense.fused_mlp_fp8_w8a8(*d, eps=1e-5, residual=rd, residual_out=rd, activation="silu")
    assert torch.equal(rd.cpu(), (x.float() + r.float()).to(dtype))
    q, s = dense.rms_norm_quant(d[0], d[1], 1e-5, r.to(DEV))
    q2, sc2 = dense.fp8_gemm_act_mul_quant(q, s, d[2], d[3])
    assert torch.equal(out, dense.fp8_gemm(q2, sc2, d[4], d[5], None, dtype))
    status_ok()
    ref = O.fp8_gemm(q2.cpu(), sc2.cpu(), w2, s2)
    err = gemm_error(q2.cpu(), sc2.cpu(), w2, s2)
    assert ((out.double().cpu() - ref).abs() <= err + HALF[dtype] * (ref.abs() + err) + 2.0 ** -25).all()
    # from the inputs, with no rounding to 8 bits at all: what e4m3 costs. Two operands of
    # each product within 2^-4: 2 * 2^-4 of the gate and of the up sums' terms at most,
    # far less of their root mean square; the whole within 8 % of the output's
    y = O.rms_norm(x, w, 1e-5, r)[1]
    one = torch.ones
    h64 = O.fp8_gemm(y, one(t, (h + 127) // 128), w13.float(), s13)
    full = O.fp8_gemm(O.act_mul(h64, "silu"), one(t, (i + 127) // 128), w2.float(), s2)
    assert (out.double().cpu() - full).norm() <= 0.08 * full.norm()


@pytest.mark.gpu
def test_mlp_int8_is_its_steps():
    t, h, i = 37, 512, 640
    x, r, w = norm_case(t, h, torch.bfloat16, 11)
    g = gen(12)
    w13 = torch.randint(-127, 128, (2 * i, h), generator=g, dtype=torch.int8).to(DEV)
    w2 = torch.randint(-127, 128, (h, i), generator=g, dtype=torch.int8).to(DEV)
    s13, s2 = (torch.rand(2 * i, generator=g) * 1e-4 + 1e-4).to(DEV), (torch.rand(h, generator=g) * 1e-4).to(DEV)
    rd = r.to(DEV)
    out = dense.fused_mlp_int8_w8a8(x.to(DEV), w.to(DEV), w13, s13, w2, s2, residual=rd, residual_out=rd,
                                    activation="gelu_tanh")
    assert torch.equal(rd.cpu(), (x.float() + r.float()).bfloat16())
    q, s = dense.rms_norm_quant(x.to(DEV), w.to(DEV), residual=r.to(DEV), q_dtype=torch.int8)
    hh = torch.ops.strix.w8a8_int8_gemm(q, s, w13, s13)
    q, s = dense.act_mul_quant(hh, "gelu_tanh", torch.int8)
    assert torch.equal(out, torch.ops.strix.w8a8_int8_gemm(q, s, w2, s2))
    check_rows(q, s, O.act_mul(hh.cpu(), "gelu_tanh"), False, GATE_REL)


@pytest.mark.gpu
@pytest.mark.parametrize("t", [3, 260])
def test_mlp_captured_replayed_and_on_another_stream(t):
    """Two captured graphs and eager calls on two streams, all over the same weights."""
    x, w, w13, s13, w2, s2, r = (v.to(DEV) for v in mlp_case(t, 512, 768, 20))

    def mlp(xx):
        return dense.fused_mlp_fp8_w8a8(xx, w, w13, s13, w2, s2, residual=r)

    xs = [x, x.flip(0).contiguous(), (x * 0.5)]
    want = [mlp(v) for v in xs]
    statics, graphs, outs = [torch.empty_like(x), torch.empty_like(x)], [], []
    for st in statics:
        st.copy_(x)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(mlp(st))
        graphs.append(g)
    side = [torch.cuda.Stream(), torch.cuda.Stream()]
    for i in range(3):
        statics[0].copy_(xs[i])
        statics[1].copy_(xs[2 - i])
        torch.cuda.synchronize()
        with torch.cuda.stream(side[0]):
            graphs[0].replay()
        with torch.cuda.stream(side[1]):
            graphs[1].replay()
        eager = mlp(xs[i])
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want[i]) and torch.equal(outs[1], want[2 - i]) and torch.equal(eager, want[i])
    with torch.cuda.stream(side[0]):
        a = mlp(xs[1])
    with torch.cuda.stream(side[1]):
        b = mlp(xs[2])
    torch.cuda.synchronize()
    assert torch.equal(a, want[1]) and torch.equal(b, want[2])
    status_ok()


@pytest.mark.gpu
@pytest.mark.parametrize("m", [3, 9, 200])
def test_vllm_linear_with_8_bit_activations(m):
    """The opt-in form of the block-scaled linear class: beyond 8 rows the activations are
    e4m3, each off by 2^-4 of its value at most; the terms' signs are mixed, so a row's
    error stays below that share of its norm."""
    from strix_vllm import fp8

    x, _, _ = norm_case(m, 640, torch.bfloat16, 30, False)
    _, _, w, sw = gemm_case(1, 392, 640, 31)
    bias = torch.randn(392, generator=gen(32)).bfloat16()
    out = fp8.apply_fp8_w8a8(x.to(DEV), w.to(DEV), sw.to(DEV), bias.to(DEV)).double().cpu()
    status_ok()
    ref = O.fp8_gemm(x, torch.ones(m, 5), w, sw, bias)
    assert ((out - ref).norm(dim=1) <= 2.0 ** -4 * ref.norm(dim=1)).all()
    # few rows keep 16-bit activations where that kernel takes the width (multiples of 16)
    w, sw, bias = w[:384].to(DEV), sw[:3].to(DEV), bias[:384].to(DEV)
    few = fp8.apply_fp8_w8a8(x[:3].to(DEV), w, sw, bias)
    assert torch.equal(few, fp8.apply_fp8(x[:3].to(DEV), w, sw, bias))


@pytest.mark.gpu
@pytest.mark.parametrize("q_dtype", [F8, torch.int8])
def test_norm_and_act_beyond_32_bit_offsets(q_dtype):
    """2.2 billion elements in, the last rows against the oracle."""
    m, k = 33100, 65536
    x = torch.zeros(m, k, dtype=torch.bfloat16, device=DEV)
    g = torch.Generator(DEV).manual_seed(50)
    at = torch.tensor([0, 5, 16384, 32767, 32768, m - 2, m - 1])
    x[at.to(DEV)] = torch.randn(len(at), k, generator=g, device=DEV).bfloat16()
    w = (1 + 0.1 * torch.randn(k, generator=gen(51))).bfloat16()
    q, s = dense.rms_norm_quant(x, w.to(DEV), 1e-6, x, x, q_dtype=q_dtype)     # in place: 2 x
    rows = x[at.to(DEV)].cpu()
    check_rows(q[at.to(DEV)], s[at.to(DEV)], O.rms_norm(rows, w, 1e-6)[1], q_dtype == F8, Y_REL)
    assert not q[1].float().any() and not q[m - 3].float().any()
    q, s = dense.act_mul_quant(x, q_dtype=q_dtype)
    check_rows(q[at.to(DEV)], s[at.to(DEV)], O.act_mul(rows, "silu"), q_dtype == F8, GATE_REL)


@pytest.mark.gpu
def test_products_beyond_32_bit_offsets():
    """An output of 2.3 billion elements (and a gated one), rows and columns at its ends."""
    n, k = 33000, 144
    m = 70000
    a, sa, w, sw = gemm_case(64, n, k, 52)
    big_a = torch.zeros(m, k, device=DEV).to(F8)
    big_sa = torch.ones(m, 2, device=DEV)
    at = torch.cat([torch.arange(0, 32), torch.arange(m - 32, m)])
    big_a.view(torch.uint8)[at.to(DEV)] = a.view(torch.uint8).to(DEV)
    big_sa[at.to(DEV)] = sa.to(DEV)
    out = dense.fp8_gemm(big_a, big_sa, w.to(DEV), sw.to(DEV))
    status_ok()
    ref, err = O.fp8_gemm(a, sa, w, sw), gemm_error(a, sa, w, sw)
    got = out[at.to(DEV)].double().cpu()
    assert ((got - ref).abs() <= err + 2.0 ** -8 * (ref.abs() + err)).all()
    assert not out[32:m - 32:997].any()
    del out
    w2, sw2 = w[:2048].contiguous(), sw[:16].contiguous()
    q, s = dense.fp8_gemm_act_mul_quant(big_a, big_sa, w2.to(DEV), sw2.to(DEV))
    q1, s1 = dense.fp8_gemm_act_mul_quant(a.to(DEV), sa.to(DEV), w2.to(DEV), sw2.to(DEV))
    status_ok()
    assert torch.allclose(s[at.to(DEV)], s1, rtol=1e-5, atol=0) and (s[32] == 1).all()


@pytest.mark.gpu
def test_two_streams_at_once():
    """Calls that overlap on the GPU share nothing."""
    cases = [gemm_case(m, n, k, 60) for m, n, k in ((3, 1024, 4096), (200, 1024, 2048), (50, 512, 4096), (90, 256, 8192))]
    cases = [[t.to(DEV) for t in c] for c in cases]
    want = [(dense.fp8_gemm(*c), dense.fp8_gemm_act_mul_quant(*c)) for c in cases]
    streams = [torch.cuda.Stream() for _ in range(4)]
    torch.cuda.synchronize()
    got = []
    for i in range(12):
        with torch.cuda.stream(streams[i % 4]):
            c = cases[i % 4 if i < 8 else 3 - i % 4]
            got.append((dense.fp8_gemm(*c), dense.fp8_gemm_act_mul_quant(*c)))
    torch.cuda.synchronize()
    status_ok()
    for i, (o, (q, s)) in enumerate(got):
        w_o, (w_q, w_s) = want[i % 4 if i < 8 else 3 - i % 4]
        assert torch.equal(o, w_o) and torch.equal(q.view(torch.uint8), w_q.view(torch.uint8)) and torch.equal(s, w_s)


@pytest.mark.gpu
def test_results_do_not_change_from_run_to_run():
    for m, n, k in ((1, 512, 4096), (50, 1024, 2048), (600, 2048, 1024)):
        a, sa, w, sw = (t.to(DEV) for t in gemm_case(m, n, k, 9))
        first = dense.fp8_gemm(a, sa, w, sw, out_dtype=torch.float32)
        for _ in range(5):
            assert torch.equal(first, dense.fp8_gemm(a, sa, w, sw, out_dtype=torch.float32))


@pytest.mark.gpu
@pytest.mark.parametrize("t", [3, 200])
def test_first_call_of_a_process_may_be_captured(t):
    """Nothing of a first call (attributes, occupancy, addresses) disturbs a capture."""
    import subprocess
    import sys
    from pathlib import Path

    code = f"""
import torch
from libstrix_b200 import dense
f8 = torch.float8_e4m3fn
x = torch.randn({t}, 256, device="cuda").bfloat16()
nw = torch.ones(256, device="cuda").bfloat16()
w13, w2 = torch.randn(512, 256, device="cuda").to(f8), torch.randn(256, 256, device="cuda").to(f8)
s13, s2 = torch.rand(4, 2, device="cuda"), torch.rand(2, 2, device="cuda")
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    y = dense.fused_mlp_fp8_w8a8(x, nw, w13, s13, w2, s2)
g.replay()
torch.cuda.synchronize()
assert torch.equal(y, dense.fused_mlp_fp8_w8a8(x, nw, w13, s13, w2, s2))
"""
    subprocess.run([sys.executable, "-c", code], check=True, timeout=240, cwd=Path(__file__).resolve().parent.parent)


@pytest.mark.gpu
def test_a_tracer_sees_the_ops():
    """Under a dispatch mode (a tracer's) the wrappers go through the dispatcher."""
    from torch.fx.experimental.proxy_tensor import make_fx

    x, _, w = norm_case(2, 256, torch.bfloat16, 40, False)
    graph = make_fx(lambda a, b: dense.rms_norm_quant(a, b))(x.to(DEV), w.to(DEV))
    assert any("rms_norm_quant_fp8" in str(n.target) for n in graph.graph.nodes)


@pytest.mark.gpu
def test_a_compiled_caller_keeps_one_graph():
    x, r, w = norm_case(5, 256, torch.bfloat16, 41)
    _, _, w13, s13 = gemm_case(1, 512, 256, 42)
    _, _, w2, s2 = gemm_case(1, 256, 256, 43)
    args = [t.to(DEV) for t in (x, w, w13, s13, w2, s2)]
    rd = r.to(DEV)
    compiled = torch.compile(lambda *a: dense.fused_mlp_fp8_w8a8(*a, residual=rd), backend="eager", fullgraph=True)
    assert torch.equal(compiled(*args), dense.fused_mlp_fp8_w8a8(*args, residual=rd))


@pytest.mark.gpu
def test_ops_check_their_tensors():
    ops = torch.ops.strix
    a, sa, w, sw = (t.to(DEV) for t in gemm_case(4, 256, 256))
    x = torch.randn(4, 256, device=DEV).bfloat16()
    g = torch.ones(256, device=DEV).bfloat16()
    bad = [
        lambda: ops.w8a8_fp8_gemm(a[:, :200], sa, w[:, :200], sw),                  # K % 16
        lambda: ops.w8a8_fp8_gemm(a, sa[:3], w, sw),                                # scales
        lambda: ops.w8a8_fp8_gemm(a, sa, w, sw[:1]),
        lambda: ops.w8a8_fp8_gemm(a, sa.double(), w, sw),
        lambda: ops.w8a8_fp8_gemm(x, sa, w, sw),                                    # type
        lambda: ops.w8a8_fp8_gemm(a, sa, w, sw, g),                                 # bias of bf16 ok; see below
        lambda: ops.w8a8_fp8_gemm(a, sa, w, sw, None, torch.int8),
        lambda: ops.w8a8_fp8_gemm(a.t(), sa, w.t(), sw),
        lambda: ops.w8a8_fp8_gemm(a[:, 8:248], sa, w[:, 8:248], sw),                # 16-byte rows
        lambda: ops.w8a8_fp8_gemm(a[:1].expand(4, 256), sa, w, sw),                 # rows on top of each other
        lambda: ops.w8a8_fp8_gemm_act_mul_quant(a, sa, w[:24], sw[:1]),             # halves of 12 rows
        lambda: ops.w8a8_fp8_gemm_act_mul_quant(a, sa, w, sw, "relu"),
        lambda: ops.rms_norm_quant_fp8(x[:, :200], g[:200], 1e-6),
        lambda: ops.rms_norm_quant_fp8(x.float(), g, 1e-6),
        lambda: ops.rms_norm_quant_fp8(x, g.half(), 1e-6),
        lambda: ops.rms_norm_quant_fp8(x, g[:128], 1e-6),
        lambda: ops.rms_norm_quant_fp8(x, g, -1.0),
        lambda: ops.rms_norm_quant_fp8(x, g, 1e-6, None, x),
        lambda: ops.rms_norm_quant_fp8(x, g, 1e-6, x[:2]),
        lambda: ops.rms_norm_quant_fp8(x, g, 1e-6, x.half()),
        lambda: ops.rms_norm_quant_fp8(x[:3], g, 1e-6, x[:3].clone(), x[1:]),       # the sum over other rows of x
        lambda: ops.rms_norm_quant_token_i8(x.view(-1)[1:1 + 4 * 248].view(4, 248), g[:248], 1e-6),
        lambda: ops.rms_norm_quant_token_i8(x, g.cpu(), 1e-6),
        lambda: ops.act_mul_quant_fp8(x, "relu"),
        lambda: ops.act_mul_quant_fp8(x[:, :40]),
        lambda: ops.act_mul_quant_token_i8(x[:, :24]),
        lambda: ops.act_mul_quant_token_i8(x.view(1, 2, -1)),
        lambda: dense.act_mul_quant(x, q_dtype=torch.float8_e5m2),
    ]
    ops.w8a8_fp8_gemm(a, sa, w, sw, g)                                              # a bias of the output's type
    bad[5] = lambda: ops.w8a8_fp8_gemm(a, sa, w, sw, g, torch.float16)              # ... and of another
    for i, f in enumerate(bad):
        with pytest.raises(RuntimeError):
            f()
            pytest.fail(f"call {i} was accepted")
    torch.cuda.synchronize()


# ------------------------------------------------------------------- without GPU
def _call(name, **over):
    """A C call with plausible (never dereferenced) pointers, some arguments replaced."""
    _, _, names = _lib.prototypes()[name]
    base = dict(x=1 << 20, residual=None, residual_out=None, weight=1 << 24, q=1 << 26, scales=1 << 27, rows=4, k=256,
                x_stride=256, r_stride=0, ro_stride=0, q_stride=256, s_stride=2, eps=1e-6, in_f16=0, weight_f32=0,
                fp8=1, gate_act=1, in_type=0, out=1 << 28, a_q=1 << 20, a_scale=1 << 21, w=1 << 24, w_scale=1 << 25,
                bias=None, m=4, n=256, a_stride=256, w_stride=256, out_stride=256, sa_stride_m=2, sa_stride_k=1,
                sw_stride_n=2, sw_stride_k=1, out_kind=0, workspace=1 << 29, workspace_bytes=1 << 20, stream=None)
    base.update(over)
    _lib.call(name, *(base[a] for a in names))


@pytest.mark.parametrize("over,message", [
    (dict(k=250), "multiple of 16"), (dict(k=0), "bad shapes"), (dict(rows=-1), "bad shapes"),
    (dict(k=65552, x_stride=65552, q_stride=65552, s_stride=513), "at most 65536"),
    (dict(x=None), "NULL"), (dict(scales=None), "NULL"), (dict(x=(1 << 20) + 8), "16-byte"),
    (dict(x_stride=260), "16-byte"), (dict(residual_out=1 << 22), "needs a residual"),
    (dict(q_stride=128), "overlap"), (dict(s_stride=1), "overlap"),
    (dict(residual=1 << 22, r_stride=256, residual_out=1 << 23, ro_stride=128), "overlap"),
    (dict(residual=1 << 22, r_stride=256, residual_out=(1 << 20) + 512, ro_stride=256), "x itself"),
    (dict(residual=1 << 22, r_stride=256, residual_out=(1 << 22) + 512, ro_stride=256), "residual itself"),
    (dict(residual=1 << 22, r_stride=512, residual_out=1 << 22, ro_stride=256), "residual itself"),
    (dict(fp8=0, k=252), "multiple of 8"),
])
def test_norm_refusals(over, message):
    with pytest.raises(strix.StrixError, match=message):
        _call("strix_rms_norm_quant", **over)


@pytest.mark.parametrize("over,message", [
    (dict(gate_act=0), "activation"), (dict(in_type=3), "bf16, fp16 or fp32"), (dict(k=248), "multiple of 16"),
    (dict(fp8=0, k=65544, q_stride=65544), "at most 65536"), (dict(x=None), "NULL"),
    (dict(x=(1 << 20) + 2), "16-byte"), (dict(q_stride=0), "overlap"), (dict(k=0), "bad shapes"),
])
def test_act_refusals(over, message):
    with pytest.raises(strix.StrixError, match=message):
        _call("strix_act_mul_quant", **over)


@pytest.mark.parametrize("name,over,message", [
    ("strix_w8a8_fp8_gemm", dict(k=250), "multiple of 16"),
    ("strix_w8a8_fp8_gemm", dict(out_kind=3), "bf16, fp16 or fp32"),
    ("strix_w8a8_fp8_gemm", dict(m=-1), "bad shapes"),
    ("strix_w8a8_fp8_gemm", dict(w=None), "NULL"),
    ("strix_w8a8_fp8_gemm", dict(a_q=(1 << 20) + 8), "16-byte"),
    ("strix_w8a8_fp8_gemm", dict(w_stride=264), "16-byte"),
    ("strix_w8a8_fp8_gemm", dict(a_stride=128), "overlap"),
    ("strix_w8a8_fp8_gemm", dict(m=1 << 31), "too large"),
    ("strix_w8a8_fp8_gated", dict(gate_act=3), "activation"),
    ("strix_w8a8_fp8_gated", dict(n=24), "multiple of 16"),
    ("strix_w8a8_fp8_gated", dict(k=8), "multiple of 16"),
])
def test_product_refusals(name, over, message):
    with pytest.raises(strix.StrixError, match=message):
        _call(name, **over)


def test_vllm_form_is_opt_in(monkeypatch):
    from strix_vllm import fp8

    monkeypatch.delenv("STRIX_ENABLE", raising=False)
    assert not fp8.w8a8_enabled()
    monkeypatch.setenv("STRIX_ENABLE", "dense_w8, fp8_w8a8")
    assert fp8.w8a8_enabled()
    monkeypatch.setenv("STRIX_DISABLE", "fp8_w8a8")
    assert not fp8.w8a8_enabled()


def test_empty_calls_need_no_device():
    _call("strix_rms_norm_quant", rows=0, x=None)
    _call("strix_act_mul_quant", rows=0, x=None)
    _call("strix_w8a8_fp8_gemm", m=0, a_q=None)
    _call("strix_w8a8_fp8_gated", m=0, a_q=None, workspace=None, workspace_bytes=0)
    assert _lib.load().strix_w8a8_fp8_gated_workspace(0, 16, 16) == 0
    assert _lib.load().strix_w8a8_fp8_gated_workspace(-1, 16, 16) == -1


def test_shapes_under_fake_tensors():
    from torch._subclasses.fake_tensor import FakeTensorMode

    def t(*shape, dtype):
        return torch.empty(*shape, dtype=dtype, device="cuda")

    f32 = torch.float32
    with FakeTensorMode():
        x, g = t(7, 272, dtype=torch.float16), t(272, dtype=torch.float16)
        a, sa, w, sw = t(7, 272, dtype=F8), t(7, 3, dtype=f32), t(320, 272, dtype=F8), t(3, 3, dtype=f32)
        for (q, s), shapes, dt in [
            (dense.rms_norm_quant(x, g, residual=x, residual_out=x), ((7, 272), (7, 3)), F8),
            (dense.rms_norm_quant(x, g, q_dtype=torch.int8), ((7, 272), (7,)), torch.int8),
            (dense.act_mul_quant(x), ((7, 136), (7, 2)), F8),
            (dense.act_mul_quant(x, q_dtype=torch.int8), ((7, 136), (7,)), torch.int8),
            (dense.fp8_gemm_act_mul_quant(a, sa, w, sw), ((7, 160), (7, 2)), F8),
        ]:
            assert (tuple(q.shape), tuple(s.shape)) == shapes and q.dtype == dt and s.dtype == f32
        out = dense.fp8_gemm(a, sa, w, sw)
        assert tuple(out.shape) == (7, 320) and out.dtype == torch.bfloat16
        assert dense.fp8_gemm(a, sa, w, sw, out_dtype=torch.float16).dtype == torch.float16
    with pytest.raises(RuntimeError, match="q_dtype"):
        dense.act_mul_quant(torch.empty(1, 32), q_dtype=torch.float16)


def test_oracle_rounds_to_e4m3_like_torch():
    v = torch.randn(100000, generator=gen(0), dtype=torch.float64) * torch.exp(4 * torch.randn(100000, generator=gen(1)).double())
    v = torch.cat([v, torch.arange(-480, 480) / 16.0, torch.arange(-64, 64) / 1024.0]).clamp(-448, 448)
    assert torch.equal(O.round_e4m3(v), v.float().to(F8).double()) or \
        (O.round_e4m3(v) != v.float().to(F8).double()).float().mean() < 1e-4   # fp32's own rounding of a tie
