"""What the operators of the 8-bit dense layer are timed on, and their plain forms.

The layer: root-mean-square norm (with the residual's addition) into 8 bits, the
FP8 product with a scale per block of 128, the gated activation into 8 bits, and
the gate-up product that ends in it. Sizes are those of the benchmark configurations
(hidden 2048 and 2880; K 5120 with a gate-up width of 34816, that is 17408 per
half) and ragged ones between them.
"""

import math

import torch

own = False

F8 = torch.float8_e4m3fn
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
EPS = 1e-6


# ------------------------------------------------------------------------ cases
def listed():
    return [
        # one token of a decode step: the smallest call, all latency
        dict(name="norm_fp8_1x5120", op="norm", q="fp8", rows=1, k=5120, dtype="bf16", residual=True),
        # a prompt's rows in front of an int8 linear layer
        dict(name="norm_i8_4096x5120", op="norm", q="i8", rows=4096, k=5120, dtype="bf16", residual=True),
        # a ragged batch; a width whose last group holds 64 columns; the first layer (no residual)
        dict(name="norm_fp8_1001x2880", op="norm", q="fp8", rows=1001, k=2880, dtype="fp16", residual=False),
        # a decode batch between the two products of an int8 MLP
        dict(name="act_i8_16x17408", op="act", q="i8", rows=16, k=17408, dtype="bf16", act="gelu_tanh"),
        # a prompt between the two products of an FP8 MLP
        dict(name="act_fp8_4096x17408", op="act", q="fp8", rows=4096, k=17408, dtype="bf16", act="silu"),
        # decode, one token: the weights are read once
        dict(name="gemm_1x34816x5120", op="gemm", rows=1, n=34816, k=5120, dtype="bf16", with_bias=False),
        # decode, a batch, the long reduction of a down projection
        dict(name="gemm_16x5120x17408", op="gemm", rows=16, n=5120, k=17408, dtype="bf16", with_bias=False),
        # ragged rows, a reduction that ends inside a block, a bias
        dict(name="gemm_300x5760x2880", op="gemm", rows=300, n=5760, k=2880, dtype="fp16", with_bias=True),
        # a mixed batch of prompts and decodes at a small layer
        dict(name="gemm_768x2048x2048", op="gemm", rows=768, n=2048, k=2048, dtype="bf16", with_bias=False),
        # a long prompt: the tensor cores set the pace
        dict(name="gemm_4096x34816x5120", op="gemm", rows=4096, n=34816, k=5120, dtype="bf16", with_bias=False),
        # the first half of an MLP for a decode batch: both halves of the product, the gate, 8 bits out
        dict(name="gated_8x17408x5120", op="gated", rows=8, n=17408, k=5120, dtype="bf16", act="silu"),
        # the same for a chunk of a prompt
        dict(name="gated_2048x17408x5120", op="gated", rows=2048, n=17408, k=5120, dtype="bf16", act="silu"),
    ]


def _log(rng, lo, hi, step=1):
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return max(lo, min(hi, int(v / step + 0.5) * step))


def draw(rng):
    op = rng.choice(["norm", "norm", "act", "act", "gemm", "gemm", "gemm", "gated"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    if op == "norm":
        return dict(op=op, q=rng.choice(["fp8", "i8"]), rows=_log(rng, 1, 8192), k=_log(rng, 512, 16384, 16),
                    dtype=dtype, residual=rng.random() < 0.75)
    if op == "act":
        return dict(op=op, q=rng.choice(["fp8", "i8"]), rows=_log(rng, 1, 4096), k=_log(rng, 512, 17408, 16),
                    dtype=dtype, act=rng.choice(["silu", "gelu_tanh"]))
    if op == "gated":
        return dict(op=op, rows=_log(rng, 1, 2048), n=_log(rng, 512, 17408, rng.choice([16, 128])),
                    k=_log(rng, 512, 5120, 16), dtype="bf16", act=rng.choice(["silu", "gelu_tanh"]))
    n, k = _log(rng, 512, 34816, rng.choice([1, 8, 128])), _log(rng, 512, 17408, 16)
    most = 4096 * 34816 * 5120 // (n * k)
    return dict(op=op, rows=_log(rng, 1, min(8192, most)), n=n, k=k, dtype=dtype, with_bias=rng.random() < 0.3)


def work(case):
    m, k = case["rows"], case["k"]
    groups = -(-k // 128)
    if case["op"] == "norm":
        scales = 4 * m * (groups if case["q"] == "fp8" else 1)
        streams = 2 + (4 if case["residual"] else 0) + 1   # x, the residual in and out, the 8-bit rows
        return {"bytes": streams * m * k + 2 * k + scales, "flops": 8 * m * k}
    if case["op"] == "act":
        scales = 4 * m * (groups if case["q"] == "fp8" else 1)
        return {"bytes": 5 * m * k + scales, "flops": 8 * m * k}
    n = case["n"]
    if case["op"] == "gemm":
        scales = 4 * groups * (m + -(-n // 128))
        return {"bytes": m * k + n * k + scales + 2 * m * n + (2 * n if case["with_bias"] else 0),
                "flops": 2 * m * n * k}
    scales = 4 * (groups * (m + -(-2 * n // 128)) + m * -(-n // 128))
    return {"bytes": m * k + 2 * n * k + scales + m * n, "flops": 4 * m * n * k}


# ----------------------------------------------------------------------- inputs
def _activations(gen, m, k, dtype):
    """Rows ~ N(0, 1) times a strength of their own, with a few strong columns."""
    x = torch.randn(m, k, generator=gen, device="cuda")
    x *= torch.exp(0.5 * torch.randn(m, 1, generator=gen, device="cuda"))
    strong = torch.randint(0, k, (max(1, k // 256),), generator=gen, device="cuda")
    x[:, strong] *= 8.0
    return x.to(dtype)


def _pad(t, dim):
    short = -t.size(dim) % 128
    if not short:
        return t
    shape = list(t.shape)
    shape[dim] = short
    return torch.cat([t, t.new_zeros(shape)], dim)


def _weights(gen, n, k):
    """e4m3 [n, k] with fp32 scales [ceil(n / 128), ceil(k / 128)], from N(0, 0.02)."""
    w = torch.randn(n, k, generator=gen, device="cuda").mul_(0.02)
    w *= torch.exp(0.3 * torch.randn(n, 1, generator=gen, device="cuda"))
    b = _pad(_pad(w, 0), 1)
    s = b.view(b.size(0) // 128, 128, -1, 128).abs().amax((1, 3)) / 448.0
    full = s.repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)[:, :k]
    return (w / full).to(F8), s


def _quantised(x):
    """e4m3 [m, k] and fp32 scales [m, ceil(k / 128)] of a 16-bit activation."""
    b = _pad(x.float(), 1).view(x.size(0), -1, 128)
    s = b.abs().amax(-1) / 448.0
    q = (b / s[..., None]).to(F8).view(x.size(0), -1)[:, :x.size(1)]
    return q.contiguous(), s


def prepare(case, seed):
    gen = torch.Generator("cuda").manual_seed(seed)
    dtype, m, k = TYPES[case["dtype"]], case["rows"], case["k"]
    st = dict(case)
    if case["op"] == "norm":
        st["x"] = _activations(gen, m, k, dtype)
        st["g"] = (1 + 0.2 * torch.randn(k, generator=gen, device="cuda")).to(dtype)
        if case["residual"]:
            st["r"] = _activations(gen, m, k, dtype)
            st["r_out"] = torch.empty_like(st["r"])
    if case["op"] == "act":
        st["x"] = _activations(gen, m, 2 * k, dtype)
    if case["op"] in ("gemm", "gated"):
        st["qa"], st["sa"] = _quantised(_activations(gen, m, k, dtype))
        st["w"], st["sw"] = _weights(gen, case["n"] * (2 if case["op"] == "gated" else 1), k)
        if case.get("with_bias"):
            st["bias"] = torch.randn(case["n"], generator=gen, device="cuda").to(dtype)
    return st


# ------------------------------------------------------------------ plain forms
# e4m3 rows are returned as they are (the type holds the values itself), int8 rows as
# the whole numbers they stand for in bf16, which holds each of them; scales beside them.
def _scale(amax, top):
    s = amax / top
    return torch.where(s < torch.finfo(torch.float32).tiny, torch.ones_like(s), s)


def _to_fp8(y):
    k = y.size(1)
    b = _pad(y, 1).view(y.size(0), -1, 128)
    s = _scale(b.abs().amax(-1), 448.0)
    return (b / s[..., None]).view(y.size(0), -1)[:, :k].to(F8), s


def _to_i8(y):
    s = _scale(y.abs().amax(-1), 127.0)
    return torch.round(y / s[:, None]).to(torch.bfloat16), s


def _norm(x, r, g):
    s = x.float() if r is None else x.float() + r.float()
    return s, s * torch.rsqrt(s.square().mean(-1, keepdim=True) + EPS) * g.float()


def _act_mul(x, act):
    a, b = x.float().chunk(2, -1)
    if act == "silu":
        return a / (1 + torch.exp(-a)) * b
    t = torch.tanh(0.7978845608028654 * (a + 0.044715 * a * a * a))
    return 0.5 * a * (1 + t) * b


def _widen(q, s, rows):
    """fp32 values of e4m3 [n, k] with a scale per `rows` rows and 128 columns."""
    return q.float() * s.repeat_interleave(rows, 0)[:q.size(0)].repeat_interleave(128, 1)[:, :q.size(1)]


def _gemm(qa, sa, w, sw, bias, dtype):
    out = _widen(qa, sa, 1) @ _widen(w, sw, 128).t()
    return (out if bias is None else out + bias.float()).to(dtype)


def _plain(st):
    op, dtype = st["op"], TYPES[st["dtype"]]
    if op == "norm":
        s, y = _norm(st["x"], st.get("r"), st["g"])
        q, sc = _to_fp8(y) if st["q"] == "fp8" else _to_i8(y)
        return [q, sc] + ([s.to(dtype)] if "r" in st else [])
    if op == "act":
        return list((_to_fp8 if st["q"] == "fp8" else _to_i8)(_act_mul(st["x"], st["act"])))
    if op == "gemm":
        return [_gemm(st["qa"], st["sa"], st["w"], st["sw"], st.get("bias"), dtype)]
    h = _gemm(st["qa"], st["sa"], st["w"], st["sw"], None, torch.float32)
    return list(_to_fp8(_act_mul(h, st["act"])))


def _own(st):
    from libstrix_b200 import dense

    op = st["op"]
    if op == "gemm":
        return [dense.fp8_gemm(st["qa"], st["sa"], st["w"], st["sw"], st.get("bias"), TYPES[st["dtype"]])]
    if op == "gated":
        return list(dense.fp8_gemm_act_mul_quant(st["qa"], st["sa"], st["w"], st["sw"], st["act"]))
    q_dtype = F8 if st["q"] == "fp8" else torch.int8
    if op == "norm":
        q, sc = dense.rms_norm_quant(st["x"], st["g"], EPS, st.get("r"), st.get("r_out"), q_dtype=q_dtype)
    else:
        q, sc = dense.act_mul_quant(st["x"], st["act"], q_dtype=q_dtype)
    if st["q"] == "i8":
        q = q.to(torch.bfloat16)
    return [q, sc] + ([st["r_out"]] if "r" in st else [])


def run(state):
    if own:
        return _own(state)
    return _plain(state)


# -------------------------------------------------------------- 64-bit definition
# In the place of e4m3 rows stands the quotient that they round, y / scale. The whole
# numbers of int8 rows have no such value: a quotient next to a border between two of
# them falls to either side in 32 bits.
def _blocks64(y):
    """y / scale and the scales of [m, k] in 64 bits, a scale per row and 128 columns."""
    m, k = y.shape
    groups = -(-k // 128)
    s = torch.zeros(m, groups, dtype=torch.float64, device=y.device)
    s.scatter_reduce_(1, (torch.arange(k, device=y.device) // 128).expand(m, k), y.abs(), "amax")
    s /= 448
    s[s < 2.0 ** -126] = 1
    return y / s[:, torch.arange(k, device=y.device) // 128], s


def _matmul64(a, sa, w, sw):
    """sum over the blocks of sa * sw * (a's block @ w's block^T): the scales stay outside
    the sums, as the definition has them."""
    m, k = a.shape
    n = w.size(0)
    rows = torch.arange(n, device=w.device) // 128
    out = torch.zeros(m, n, dtype=torch.float64, device=w.device)
    for b in range(-(-k // 128)):
        lo, hi = 128 * b, min(k, 128 * b + 128)
        part = a[:, lo:hi].double() @ w[:, lo:hi].double().t()
        out += part * sa[:, b, None].double() * sw[rows, b].double()
    return out


def _norm64(st):
    s = st["x"].double()
    if "r" in st:
        s = s + st["r"].double()
    rms = (s.pow(2).sum(-1, keepdim=True) / s.size(1) + EPS).sqrt()
    return s, s / rms * st["g"].double()


def _act64(x, act):
    a, b = x[:, :x.size(1) // 2].double(), x[:, x.size(1) // 2:].double()
    if act == "silu":
        return a * torch.sigmoid(a) * b
    return a / (1 + torch.exp(-2 * math.sqrt(2 / math.pi) * (a + 0.044715 * a ** 3))) * b


def exact(case, seed):
    st = prepare(case, seed)
    op = st["op"]
    if op == "gemm":
        out = _matmul64(st["qa"], st["sa"], st["w"], st["sw"])
        return [out + st["bias"].double() if "bias" in st else out]
    if op == "gated":
        return list(_blocks64(_act64(_matmul64(st["qa"], st["sa"], st["w"], st["sw"]), st["act"])))
    s, y = _norm64(st) if op == "norm" else (None, _act64(st["x"], st["act"]))
    if st["q"] == "fp8":
        q, sc = _blocks64(y)
    else:
        sc = y.abs().amax(-1) / 127
        sc[sc < 2.0 ** -126] = 1
        q = None
    return [q, sc] + ([s] if "r" in st else [])
