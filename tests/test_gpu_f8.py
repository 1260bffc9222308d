"""The 8-bit float operators on a GPU against their definitions in 64 bits
(f8_ref.py derives the tolerances), over types, sizes that end inside blocks
and tiles, row strides, masks, empty groups, streams and graphs."""
from __future__ import annotations

import threading

import pytest
import torch

import f8_ref as R
from futon_b200 import FutonError, _lib, f8

pytestmark = pytest.mark.gpu

F8 = torch.float8_e4m3fn
TYPES = [torch.float32, torch.float16, torch.bfloat16]


@pytest.fixture(autouse=True)
def clean(gpu):
    """Every test ends with the device having found nothing."""
    yield
    f8.f8_sync(0)


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def rows(g, r, k):
    """Rows of different sizes with a few loud columns."""
    x = torch.randn(r, k, generator=g, device="cuda")
    x *= torch.exp(torch.randn(r, 1, generator=g, device="cuda"))
    return x * torch.where(torch.rand(k, generator=g, device="cuda") < 0.02, 20.0, 1.0)


# ---- quantisation ---------------------------------------------------------

SHAPES = [(1, 1), (1, 128), (3, 129), (5, 384), (2, 127), (33, 1000), (17, 4096), (1, 5001), (300, 8)]


def act_exact(x, act):
    y = x.double()
    if act == "gelu":
        return y * torch.special.erfc(-y / 2 ** 0.5) / 2, R.Y_GELU
    if act == "swiglu":
        up, gate = y.chunk(2, 1)
        return up * gate * torch.sigmoid(gate), R.Y_SWIGLU
    return y, R.Y_NONE


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("act", ["none", "gelu", "swiglu"])
@pytest.mark.parametrize("r,k", SHAPES)
def test_quantize_rows(dtype, act, r, k):
    g = gen(r * 10007 + k)
    x = rows(g, r, 2 * k if act == "swiglu" else k)
    if act == "gelu":
        x = x.clamp(-6, 6)
    if act == "swiglu":
        x[:, k:] = x[:, k:].clamp(-40, 40)
    x = x.to(dtype)
    q, s = f8.quantize_f8(x, activation=act)
    assert q.shape == (r, k) and q.dtype == F8 and s.shape == (r, -(-k // 128))
    y, rel = act_exact(x, act)
    R.check_quantised(y, q, s, 1, rel)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("r,k", [(1, 1), (128, 128), (127, 129), (129, 127), (300, 1000), (1, 500), (513, 8)])
def test_quantize_tiles(dtype, r, k):
    x = rows(gen(r + k), r, k).to(dtype)
    q, s = f8.quantize_f8(x, block_rows=128)
    R.check_quantised(x.double(), q, s, 128, R.Y_NONE)


@pytest.mark.parametrize("act", ["none", "swiglu"])
@pytest.mark.parametrize("shift,pad", [(0, 8), (1, 0), (3, 5), (0, 1)])
def test_quantize_strides(act, shift, pad):
    """Rows that start anywhere give the codes of contiguous ones; room
    between the output's rows stays as it was."""
    r, k = 7, 333
    w = 2 * k if act == "swiglu" else k
    x = rows(gen(5), r, w).half()
    room = torch.full((r * (w + pad) + shift,), float("nan"), dtype=torch.float16, device="cuda")
    xs = room[shift:].view(r, w + pad)[:, :w]
    xs.copy_(x)
    out = torch.full((r, k + 3), 0x55, dtype=torch.uint8, device="cuda")
    q, s = f8.quantize_f8(xs, activation=act,
                          out=(out.view(F8)[:, :k], torch.empty(r, 3, device="cuda")))
    q0, s0 = f8.quantize_f8(x, activation=act)
    assert torch.equal(q.view(torch.uint8), q0.view(torch.uint8)) and torch.equal(s, s0)
    assert (out[:, k:] == 0x55).all()


@pytest.mark.parametrize("block_rows", [1, 128])
def test_quantize_edges(block_rows):
    """Zero blocks, the least scale, ties, the largest value, NaN and infinity
    stay inside their own block."""
    x = torch.randn(256, 512, generator=gen(3), device="cuda")
    x[:128, :128] = 0.0
    x[0, 128:256] = float("nan")
    x[1, 256] = float("inf")
    x[2, 384:] = 2.0 ** -126
    x[130, 0:8] = torch.tensor([448.0, 17.0, 19.0, -17.0, 0.0, -0.0, 1.0, 2.0 ** -9 * 1.5])
    q, s = f8.quantize_f8(x, block_rows=block_rows)
    y = x.double()
    if block_rows == 1:
        assert s[0, 0] == 2.0 ** -100 / 448 and (q[:128, :128].float() == 0).all()
        assert s[0, 1].isnan() and q[0, 128:256].float().isnan().all()
        assert s[1, 2].isinf() and q[1, 256].float().isnan() and (q[1, 257:384].float() == 0).all()
        assert s[2, 3] == 2.0 ** -100 / 448 and (q[2, 384:].float() == 0).all()
        # 448 maps to 448, and 17 and 19 lie half-way between codes 16, 18 and 20.
        x[130, 8:128] = 0.0
        q2, s2 = f8.quantize_f8(x[130:131, :128].contiguous())
        assert s2[0, 0] == 1.0
        assert q2[0, :7].float().tolist() == [448.0, 16.0, 20.0, -16.0, 0.0, 0.0, 1.0]
        assert q2[0, 7].float() == 2.0 ** -9 * 2  # a tie between subnormals goes to the even one
    else:
        assert s.shape == (2, 4)
        assert s[0, 0] == 2.0 ** -100 / 448 and (q[:128, :128].float() == 0).all()
        assert s[0, 1].isnan() and q[:128, 128:256].float().isnan().all()
        assert s[0, 2].isinf() and q[1, 256].float().isnan() and (q[2:128, 256:384].float() == 0).all()
        R.check_quantised(y[128:], q[128:], s[1:], 128, R.Y_NONE)


# ---- RMS norm -------------------------------------------------------------

def norm_exact(x, res, w, eps):
    h = x.double() if res is None else x.double() + res.double()
    y = h / torch.sqrt((h * h).mean(1, keepdim=True) + eps) * w.double()
    return h, y


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("r,k", [(1, 1), (1, 4096), (2, 130), (600, 8), (400, 384), (333, 768), (9, 1024),
                                 (700, 1000), (300, 2056), (500, 4096), (3, 5000), (5, 9001),
                                 (2, 16384), (3, 20000), (350, 1025)])
def test_rms_norm(dtype, residual, r, k):
    g = gen(r * 31 + k)
    x = rows(g, r, k).to(dtype)
    res = torch.randn(r, k, generator=g, device="cuda").to(dtype) if residual else None
    w = 1 + 0.1 * torch.randn(k, generator=g, device="cuda")
    q, s, h = f8.rms_norm_f8(x, w, 1e-6, residual=res)
    he, y = norm_exact(x, res, w, 1e-6)
    R.check_quantised(y, q, s, 1, R.Y_NORM)
    if residual:
        # One f32 sum of two values of the type, then one rounding.
        assert h.dtype == dtype
        half = torch.finfo(dtype).eps / 2 + 2.0 ** -24
        assert ((h.double() - he).abs() <= he.abs() * half * (1 + 2.0 ** -20) + 2.0 ** -25).all()
        assert torch.equal(h, (x.float() + res.float()).to(dtype))
    else:
        assert h is None


@pytest.mark.parametrize("r,k", [(4, 768), (3, 20000), (400, 333)])
@pytest.mark.parametrize("over", ["residual", "x"])
def test_rms_norm_in_place(r, k, over):
    """residual_out over the residual, or over x."""
    g = gen(k)
    x, res = rows(g, r, k).half(), torch.randn(r, k, generator=g, device="cuda").half()
    w = torch.ones(k, device="cuda")
    q0, s0, h0 = f8.rms_norm_f8(x, w, 1e-5, residual=res)
    x1, r1 = x.clone(), res.clone()
    q, s, h = f8.rms_norm_f8(x1, w, 1e-5, residual=r1, residual_out=r1 if over == "residual" else x1)
    assert torch.equal(h, h0) and torch.equal(s, s0)
    assert torch.equal(q.view(torch.uint8), q0.view(torch.uint8))
    assert torch.equal(x1 if over == "residual" else r1, x if over == "residual" else res)


def test_rms_norm_stores_x_without_a_residual():
    x = rows(gen(2), 5, 200).bfloat16()
    out = torch.zeros_like(x)
    f8.rms_norm_f8(x, torch.ones(200, device="cuda"), 0.0, residual_out=out)
    assert torch.equal(out, x)


def test_rms_norm_strides_and_zero_rows():
    r, k = 6, 450
    g = gen(8)
    x = rows(g, r, k + 7)[:, 3:k + 3]
    res = torch.randn(r, k + 1, generator=g, device="cuda")[:, :k]
    x[2] = 0
    res[2] = 0
    w = torch.randn(k + 1, generator=g, device="cuda")[1:]  # not at a multiple of 16 bytes
    q, s, h = f8.rms_norm_f8(x, w.contiguous(), 1e-6, residual=res)
    q1, s1, h1 = f8.rms_norm_f8(x.contiguous(), w.contiguous().clone(), 1e-6, residual=res.contiguous())
    assert torch.equal(q.view(torch.uint8), q1.view(torch.uint8)) and torch.equal(s, s1) and torch.equal(h, h1)
    assert (q[2].float() == 0).all() and (s[2] == 2.0 ** -100 / 448).all()
    x[4, 5] = float("nan")
    q, s, _ = f8.rms_norm_f8(x, w.contiguous(), 1e-6, residual=res)
    assert s[4].isnan().all() and not s[[0, 1, 2, 3, 5]].isnan().any()


# ---- block-scaled product -------------------------------------------------

def product_inputs(g, m, n, k):
    aq, sa = R.quantised(rows(g, m, k), 1)
    bq, sb = R.quantised(0.02 * torch.randn(n, k, generator=g, device="cuda"), 128)
    return R.pitched(aq), sa, R.pitched(bq), sb


def check_f8(got, aq, sa, bq, sb, bias, k):
    a, b = R.values(aq, sa, 1), R.values(bq, sb, 128)
    want, mag = a @ b.t(), a.abs() @ b.abs().t()
    if bias is not None:
        want, mag = want + bias.double(), mag + bias.double().abs()
    R.check_product(got, want, mag, k)


PRODUCTS = [(1, 1, 1), (1, 128, 128), (1, 4096, 4096), (7, 129, 100), (16, 200, 384), (17, 384, 1536),
            (33, 1152, 384), (64, 100, 16), (65, 256, 128), (128, 256, 256), (130, 257, 300),
            (200, 1000, 777), (500, 513, 129), (1000, 2304, 768), (2500, 384, 1536), (3, 7, 8200),
            (64, 130, 5000), (257, 4096, 64)]


@pytest.mark.parametrize("m,n,k", PRODUCTS)
@pytest.mark.parametrize("dtype", TYPES)
def test_matmul_f8(m, n, k, dtype):
    g = gen(m * 7 + n * 3 + k)
    aq, sa, bq, sb = product_inputs(g, m, n, k)
    bias = torch.randn(n, generator=g, device="cuda") if (m + n + k) % 2 else None
    got = f8.matmul_t_f8(aq, sa, bq, sb, bias=bias, out_dtype=dtype)
    assert got.dtype == dtype and got.shape == (m, n)
    check_f8(got, aq, sa, bq, sb, bias, k)


@pytest.mark.parametrize("m", [5, 50, 300])
def test_matmul_f8_exact_sums(m):
    """Small whole numbers: every sum is exact in f32, so every element of
    every tile has to be right to the bit."""
    n, k = 390, 1000
    g = gen(m)
    a = torch.randint(-8, 9, (m, k), generator=g, device="cuda").float()
    b = torch.randint(-8, 9, (n, k), generator=g, device="cuda").float()
    sa = 2.0 ** torch.randint(-3, 4, (m, 8), generator=g, device="cuda").float()
    sb = 2.0 ** torch.randint(-3, 4, (4, 8), generator=g, device="cuda").float()
    aq, bq = R.pitched(a.to(F8)), R.pitched(b.to(F8))
    got = f8.matmul_t_f8(aq, sa, bq, sb, out_dtype=torch.float32)
    want = R.values(aq, sa, 1) @ R.values(bq, sb, 128).t()
    assert torch.equal(got.double(), want)
    # The same twice, and into a strided output whose gaps stay as they were.
    room = torch.full((m, n + 5), 7.0, device="cuda")
    f8.matmul_t_f8(aq, sa, bq, sb, out=room[:, :n])
    assert torch.equal(room[:, :n], got) and (room[:, n:] == 7).all()


@pytest.mark.parametrize("m,n,k", [(700, 1000, 300), (1100, 520, 256), (33, 260, 4096), (2050, 2049, 40)])
@pytest.mark.parametrize("dtype", TYPES)
def test_matmul_f8_output_with_room(m, n, k, dtype):
    """Rows of the output that lie further apart than n, at multiples of 16
    bytes and elsewhere: the same values, and the room stays as it was."""
    g = gen(m + n)
    aq, sa, bq, sb = product_inputs(g, m, n, k)
    bias = torch.randn(n, generator=g, device="cuda")
    want = f8.matmul_t_f8(aq, sa, bq, sb, bias=bias, out_dtype=dtype)
    check_f8(want, aq, sa, bq, sb, bias, k)
    for wide, shift in ((-(-n // 16) * 16 + 16, 0), (n + 3, 0), (-(-n // 16) * 16 + 16, 8), (n + 1, 1)):
        room = torch.full(((m + 40) * wide + shift,), 9.0, dtype=dtype, device="cuda")
        view = room[shift:].view(m + 40, wide)
        f8.matmul_t_f8(aq, sa, bq, sb, bias=bias, out=view[:m, :n])
        assert torch.equal(view[:m, :n], want)
        assert (view[:, n:] == 9).all() and (view[m:] == 9).all() and (room[:shift] == 9).all()


@pytest.mark.parametrize("m", [3, 40, 200])
def test_matmul_f8_nan_and_inf_stay_in_their_rows(m):
    n, k = 300, 300
    aq, sa, bq, sb = product_inputs(gen(m + 1), m, n, k)
    base = f8.matmul_t_f8(aq, sa, bq, sb, out_dtype=torch.float32)
    sa2, sb2 = sa.clone(), sb.clone()
    sa2[1, 1] = float("nan")
    sb2[2, 0] = float("inf")
    got = f8.matmul_t_f8(aq, sa2, bq, sb2, out_dtype=torch.float32)
    assert got[1].isnan().all()
    keep = [i for i in range(m) if i != 1]
    assert torch.equal(got[keep][:, :256], base[keep][:, :256])
    assert not got[keep][:, 256:].isfinite().any()


# ---- grouped product ------------------------------------------------------

def grouped_inputs(g, sizes, n, k, dtype, lead=0, tail=0):
    m, e = lead + sum(sizes) + tail, len(sizes)
    off = torch.tensor([lead + sum(sizes[:i]) for i in range(e + 1)], dtype=torch.int32, device="cuda")
    a = rows(g, m, k)
    w = 0.05 * torch.randn(e, n, k, generator=g, device="cuda")
    if dtype == F8:
        aq, sa = R.quantised(a, 1)
        qs = [R.quantised(w[i], 128) for i in range(e)]
        bq, sb = torch.stack([q.view(torch.uint8) for q, _ in qs]).view(F8), torch.stack([s for _, s in qs])
        av = R.values(aq, sa, 1)
        bv = torch.stack([R.values(q, s, 128) for q, s in qs])
        return R.pitched(aq), R.pitched(bq), off, sa, sb, av, bv
    a, w = a.to(dtype), w.to(dtype)
    return R.pitched(a), R.pitched(w), off, None, None, a.double(), w.double()


def check_grouped(got, before, off, av, bv, bias, k):
    o = off.tolist()
    inside = torch.zeros(got.shape[0], dtype=torch.bool)
    for i in range(len(o) - 1):
        lo, hi = o[i], o[i + 1]
        inside[lo:hi] = True
        if hi > lo:
            want, mag = av[lo:hi] @ bv[i].t(), av[lo:hi].abs() @ bv[i].abs().t()
            if bias is not None:
                want, mag = want + bias[i].double(), mag + bias[i].double().abs()
            R.check_product(got[lo:hi], want, mag, k)
    outside = (~inside).cuda()
    assert torch.equal(got[outside], before[outside])


GROUPS = [([1], 1, 8), ([0, 0, 3], 130, 100), ([5, 0, 1, 16, 17], 257, 384), ([64, 1, 0, 2], 96, 72),
          ([40, 100, 0, 30, 33], 300, 200), ([0, 300, 7, 129], 384, 1536), ([0, 0], 64, 64),
          ([1] * 70, 40, 136), ([2, 0, 0, 4000], 128, 64), ([700, 650, 0, 900], 520, 328),
          ([0] * 1000 + [9] * 24, 16, 32)]


@pytest.mark.parametrize("dtype", [F8, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("sizes,n,k", GROUPS)
def test_grouped(dtype, sizes, n, k):
    g = gen(len(sizes) + sum(sizes) + n)
    for lead, tail, bias, out in ((0, 0, False, torch.float32), (3, 5, True, torch.bfloat16),
                                  (0, 2, False, torch.float16)):
        a, b, off, sa, sb, av, bv = grouped_inputs(g, sizes, n, k, dtype, lead, tail)
        if a.shape[0] == 0:
            continue
        bv_ = torch.randn(len(sizes), n, generator=g, device="cuda") if bias else None
        got = torch.full((a.shape[0], n), 5.0, dtype=out, device="cuda")
        before = got.clone()
        r = f8.matmul_t_grouped(a, b, off, a_scales=sa, b_scales=sb, bias=bv_, out=got)
        assert r is got
        check_grouped(got, before, off, av, bv, bv_, k)


@pytest.mark.parametrize("dtype", [F8, torch.float16])
@pytest.mark.parametrize("sizes,n,k", [([17, 15] * 9, 128, 2048), ([33, 1, 0, 14] * 5, 256, 1024),
                                       ([40, 20, 36] * 4, 128, 1536), ([130, 0, 2] * 3, 100, 4096)])
def test_grouped_split_clusters_take_several_tiles(dtype, sizes, n, k):
    """Few tiles on the SMs and a long k: clusters share tiles, some take
    several, and some of their CTAs have no tokens of a tile to store. Many
    launches in a row, all the same to the bit."""
    a, b, off, sa, sb, av, bv = grouped_inputs(gen(k), sizes, n, k, dtype)
    first = f8.matmul_t_grouped(a, b, off, a_scales=sa, b_scales=sb, out_dtype=torch.float32)
    check_grouped(first, first, off, av, bv, None, k)
    outs = [f8.matmul_t_grouped(a, b, off, a_scales=sa, b_scales=sb, out_dtype=torch.float32)
            for _ in range(50)]
    assert all(torch.equal(o, first) for o in outs)


@pytest.mark.parametrize("dtype", [F8, torch.bfloat16])
@pytest.mark.parametrize("off", [[0, 9, 4, 12], [-3, 2, 5, 8], [0, 5, 40, 60], [7, 3, 1, 0]])
def test_grouped_bad_offsets_are_clamped_and_reported(dtype, off):
    sizes, n, k = [4, 4, 4], 70, 96
    a, b, _, sa, sb, av, bv = grouped_inputs(gen(1), sizes, n, k, dtype)
    bad = torch.tensor(off, dtype=torch.int32, device="cuda")
    got = torch.full((12, n), 5.0, device="cuda")
    before = got.clone()
    f8.matmul_t_grouped(a, b, bad, a_scales=sa, b_scales=sb, out=got)
    with pytest.raises(FutonError, match="offsets") as ei:
        f8.f8_sync()
    assert ei.value.code == _lib.FUTON_EDEVICE
    f8.f8_sync()  # reported once
    clamped, top = [], 0
    for v in off:
        top = max(top, min(max(v, 0), 12))
        clamped.append(top)
    check_grouped(got, before, torch.tensor(clamped), av, bv, None, k)


def test_grouped_single_row_matrices_and_padded_stack():
    """n = 1, and matrices whose rows are wider than k."""
    g = gen(4)
    for n, k, dtype in ((1, 64, torch.float16), (1, 40, F8), (5, 33, torch.bfloat16), (3, 17, F8)):
        a, b, off, sa, sb, av, bv = grouped_inputs(g, [3, 0, 4], n, k, dtype)
        got = f8.matmul_t_grouped(a, b, off, a_scales=sa, b_scales=sb, out_dtype=torch.float32)
        check_grouped(got, got, off, av, bv, None, k)


# ---- as they are used -----------------------------------------------------

def feed_forward(x, res, gamma, fc1, fc2, h):
    """Norm, fc1‖gate, SwiGLU, fc2: the feed-forward half of a block."""
    q, s, r = f8.rms_norm_f8(x, gamma, 1e-6, residual=res, residual_out=h)
    y = f8.matmul_t_f8(q, s, *fc1, out_dtype=torch.float16)
    q, s = f8.quantize_f8(y, activation="swiglu")
    return f8.matmul_t_f8(q, s, *fc2, out_dtype=torch.float16)


@pytest.mark.parametrize("m", [1, 31, 700])
def test_feed_forward_block(m):
    """The run of the operators stays near the block in 64 bits on the
    unquantised weights: each quantised operand is off by 2^-4/√3 of a value
    at most (a uniform error of half a step), independently, four times."""
    hid, mid = 384, 1536
    g = gen(m)
    x, res = rows(g, m, hid).half(), torch.randn(m, hid, generator=g, device="cuda").half()
    gamma = 1 + 0.1 * torch.randn(hid, generator=g, device="cuda")
    w1 = 0.05 * torch.randn(2 * mid, hid, generator=g, device="cuda")
    w2 = 0.05 * torch.randn(hid, mid, generator=g, device="cuda")
    fc1, fc2 = f8.quantize_f8(w1, block_rows=128), f8.quantize_f8(w2, block_rows=128)
    got = feed_forward(x, res, gamma, fc1, fc2, torch.empty_like(x))
    h, y = norm_exact(x, res, gamma, 1e-6)
    up, gate = (y @ w1.double().t()).chunk(2, 1)
    want = (up * gate * torch.sigmoid(gate)) @ w2.double().t()
    rel = ((got.double() - want).norm() / want.norm()).item()
    # up and gate each carry two operands' errors, their product both, and
    # the second product two more: √6 · 2^-4/√3 is the sum of six.
    assert rel <= 6 ** 0.5 * 2.0 ** -4 / 3 ** 0.5, rel


@pytest.mark.parametrize("tokens", [5, 400])
def test_experts_block(tokens):
    """Top-2 routing over experts: rows sorted by expert, both grouped
    products, and the weighted sum back, against each token's own experts."""
    hid, mid, e = 256, 384, 6
    g = gen(tokens)
    x = rows(g, tokens, hid).bfloat16()
    gamma = torch.ones(hid, device="cuda")
    w1 = 0.05 * torch.randn(e, 2 * mid, hid, generator=g, device="cuda")
    w2 = 0.05 * torch.randn(e, hid, mid, generator=g, device="cuda")
    p, pick = torch.randn(tokens, e, generator=g, device="cuda").softmax(1).topk(2, dim=1)
    order = pick.flatten().argsort(stable=True)
    off = torch.zeros(e + 1, dtype=torch.int32, device="cuda")
    off[1:] = torch.bincount(pick.flatten(), minlength=e).cumsum(0)
    stack = lambda w: tuple(torch.stack(t) for t in zip(*(
        (q.view(torch.uint8), s) for q, s in (f8.quantize_f8(v, block_rows=128) for v in w))))
    (b1, s1), (b2, s2) = stack(w1), stack(w2)
    q, s, _ = f8.rms_norm_f8(x, gamma, 1e-6)
    rowsel = order // 2
    y = f8.matmul_t_grouped(q.view(torch.uint8)[rowsel].view(F8), b1.view(F8), off, a_scales=s[rowsel],
                            b_scales=s1)
    q2, sc2 = f8.quantize_f8(y, activation="swiglu")
    z = f8.matmul_t_grouped(q2, b2.view(F8), off, a_scales=sc2, b_scales=s2, out_dtype=torch.float32)
    got = torch.zeros(tokens, hid, device="cuda").index_add_(0, rowsel, z * p.flatten()[order, None])
    _, yn = norm_exact(x, None, gamma, 1e-6)
    want = torch.zeros(tokens, hid, dtype=torch.float64, device="cuda")
    for t in range(tokens):
        for j in range(2):
            i = pick[t, j]
            up, gate = (w1[i].double() @ yn[t]).chunk(2)
            want[t] += p[t, j].double() * (w2[i].double() @ (up * gate * torch.sigmoid(gate)))
    rel = ((got.double() - want).norm() / want.norm()).item()
    assert rel <= 6 ** 0.5 * 2.0 ** -4 / 3 ** 0.5, rel


def test_graph_replays_with_new_inputs():
    """A captured block replays on new contents of the same buffers, and two
    graphs that interleave on two streams do not disturb one another."""
    m, hid, mid = 40, 384, 512
    g = gen(12)
    gamma = torch.ones(hid, device="cuda")
    fc1 = f8.quantize_f8(0.05 * torch.randn(2 * mid, hid, generator=g, device="cuda"), block_rows=128)
    fc2 = f8.quantize_f8(0.05 * torch.randn(hid, mid, generator=g, device="cuda"), block_rows=128)
    states = []
    for i in range(2):
        x, res = torch.empty(m, hid, device="cuda").half(), torch.empty(m, hid, device="cuda").half()
        h = torch.empty_like(x)
        st = torch.cuda.Stream()
        graph = torch.cuda.CUDAGraph()
        x.zero_(), res.zero_()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=st):
            y = feed_forward(x, res, gamma, fc1, fc2, h)
        states.append((x, res, h, y, st, graph))
    for r in range(3):
        want = []
        for x, res, h, y, st, graph in states:
            x.copy_(rows(g, m, hid)), res.copy_(rows(g, m, hid))
            h0 = torch.empty_like(x)
            want.append((feed_forward(x, res, gamma, fc1, fc2, h0), h0))
        torch.cuda.synchronize()
        for _ in range(5):
            for *_, st, graph in states:
                with torch.cuda.stream(st):
                    graph.replay()
        torch.cuda.synchronize()
        for (x, res, h, y, st, graph), (w, h0) in zip(states, want):
            assert torch.equal(y, w) and torch.equal(h, h0)


def test_streams_and_threads():
    """Calls from several host threads on streams of their own give the
    results of one thread, bit for bit."""
    cases = []
    for i, (m, n, k) in enumerate([(1, 1024, 2048), (40, 640, 1000), (300, 520, 384), (64, 4096, 256)]):
        aq, sa, bq, sb = product_inputs(gen(i), m, n, k)
        cases.append((aq, sa, bq, sb, f8.matmul_t_f8(aq, sa, bq, sb, out_dtype=torch.float32)))
    x = rows(gen(9), 500, 768).half()
    q0, s0, _ = f8.rms_norm_f8(x, torch.ones(768, device="cuda"), 1e-6)
    w = torch.ones(768, device="cuda")
    torch.cuda.synchronize()
    errors = []

    def worker(t):
        try:
            st = torch.cuda.Stream()
            with torch.cuda.stream(st):
                for r in range(20):
                    aq, sa, bq, sb, want = cases[(t + r) % 4]
                    got = f8.matmul_t_f8(aq, sa, bq, sb, out_dtype=torch.float32)
                    q, s, _ = f8.rms_norm_f8(x, w, 1e-6)
                    st.synchronize()
                    if not (torch.equal(got, want) and torch.equal(s, s0)
                            and torch.equal(q.view(torch.uint8), q0.view(torch.uint8))):
                        errors.append((t, r))
            st.synchronize()
        except Exception as e:  # noqa: BLE001 - reported below
            errors.append((t, repr(e)))

    threads = [threading.Thread(target=worker, args=(t,)) for t in range(4)]
    for th in threads:
        th.start()
    for th in threads:
        th.join(timeout=120)
    assert not any(th.is_alive() for th in threads) and not errors, errors[:4]


def test_offsets_past_32_bits():
    """Rows whose elements lie more than 2^31 from the first: the last ones
    equal those of a call on them alone (for the norm, whose sums a few rows
    add in another order, they are as near to the definition)."""
    r, k = 280_000, 8192  # 2.3e9 elements
    x = torch.zeros(r, k, dtype=torch.float16, device="cuda")
    x[-3:] = rows(gen(6), 3, k).half()
    w = torch.ones(k, device="cuda")
    q, s, _ = f8.rms_norm_f8(x, w, 1e-6)
    R.check_quantised(norm_exact(x[-3:], None, w, 1e-6)[1], q[-3:], s[-3:], 1, R.Y_NORM)
    assert (q[r // 2].float() == 0).all()
    del q, s
    for call in (lambda t: f8.quantize_f8(t), lambda t: f8.quantize_f8(t, activation="swiglu")):
        q, s = call(x)
        q1, s1 = call(x[-3:].contiguous())
        assert torch.equal(q[-3:].view(torch.uint8), q1.view(torch.uint8))
        assert torch.equal(s[-3:], s1) and (q[r // 2].float() == 0).all()
        del q, s
    del x
    m, n, k = 70_000, 32_768, 32  # 2.3e9 outputs
    aq, sa, bq, sb = product_inputs(gen(7), m, n, k)
    got = f8.matmul_t_f8(aq, sa, bq, sb)
    assert torch.equal(got[-300:], f8.matmul_t_f8(aq[-300:], sa[-300:].contiguous(), bq, sb))
    off = torch.tensor([0, 10, m - 40, m], dtype=torch.int32, device="cuda")
    b3 = bq.view(torch.uint8).expand(3, n, k).contiguous().view(F8)
    s3 = sb.expand(3, *sb.shape).contiguous()
    assert torch.equal(f8.matmul_t_grouped(aq, b3, off, a_scales=sa, b_scales=s3)[-300:], got[-300:])


def test_first_use_inside_a_capture():
    """The first call of a process may be one that is captured (the set-up is
    no stream work)."""
    import subprocess
    import sys
    code = """
import torch
from futon_b200 import f8
x = torch.randn(50, 384, device="cuda").half()
w = torch.randn(256, 384, device="cuda")
g = torch.cuda.CUDAGraph()
torch.cuda.synchronize()
with torch.cuda.graph(g):
    q, s = f8.quantize_f8(x)
    wq, ws = f8.quantize_f8(w, block_rows=128)
    y = f8.matmul_t_f8(q, s, wq, ws)
    q2, s2, _ = f8.rms_norm_f8(x, torch.ones(384, device="cuda"), 1e-6)
g.replay()
want = f8.matmul_t_f8(*f8.quantize_f8(x), *f8.quantize_f8(w, block_rows=128))
torch.cuda.synchronize()
assert torch.equal(y, want)
f8.f8_sync()
print("captured")
"""
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=120,
                       cwd=str(R.__file__).rsplit("/tests/", 1)[0])
    assert r.returncode == 0 and "captured" in r.stdout, r.stderr[-2000:]


def test_current_device_stays():
    """A call leaves the thread's current device as it was."""
    before = torch.cuda.current_device()
    f8.quantize_f8(torch.ones(2, 64, device="cuda"))
    f8.f8_sync("cuda:0")
    assert torch.cuda.current_device() == before
