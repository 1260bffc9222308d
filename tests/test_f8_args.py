"""The 8-bit float operators refuse bad arguments before any device work
(no GPU needed): the C entry points by code and message, the tensor layer by
the same error."""
from __future__ import annotations

import ctypes as C

import pytest

from futon_b200 import FutonError, _lib, f8

E = _lib.FUTON_EINVAL
P = 1 << 20  # an aligned address that a refused call never touches

QUANT = dict(dev=0, q=P, ldq=64, scales=P, src=P, lds=64, dtype=0, rows=2, k=64, act=0,
             block_rows=1, stream=None)
NORM = dict(dev=0, q=P, ldq=64, scales=P, out=None, ldo=0, x=P, ldx=64, residual=None, ldr=0, w=P,
            dtype=1, rows=2, k=64, eps=1e-6, stream=None)
MATMUL = dict(dev=0, dst=P, dst_dtype=0, ldd=8, a=P, lda=64, a_scales=P, b=P, ldb=64, b_scales=P,
              m=2, n=8, k=64, bias=None, stream=None)
GROUPED = dict(dev=0, dst=P, dst_dtype=0, ldd=8, a=P, lda=64, a_scales=None, b=P, ldb=64,
               b_scales=None, dtype=1, offsets=P, groups=3, m=2, n=8, k=64, bias=None, stream=None)


def refused(fn, base, match, **changes):
    args = dict(base, **changes)
    assert list(args) == list(base)
    with pytest.raises(FutonError, match=match) as ei:
        _lib.call(fn, *args.values())
    assert ei.value.code == E


@pytest.mark.parametrize("changes,match", [
    (dict(rows=-1), "rows=-1"), (dict(k=0), "k=0"), (dict(k=(1 << 30) + 1), "shape"),
    (dict(dtype=3), "dtype 3"), (dict(dtype=-1), "dtype -1"), (dict(act=3), "activation 3"),
    (dict(block_rows=64), "block_rows=64"), (dict(block_rows=128, act=1), "no activation"),
    (dict(ldq=63), "ldq=63"), (dict(lds=63), "lds=63"), (dict(act=2), "lds=64"),
    (dict(dev=-1), "bad device -1"), (dict(dev=64), "bad device 64"),
    (dict(q=None), "null buffer"), (dict(scales=None), "null buffer"),
    (dict(src=None), "null buffer"), (dict(src=P + 2), "misaligned"),
    (dict(scales=P + 1), "misaligned"),
])
def test_quantize_refusals(changes, match):
    refused("futon_cuda_quantize_f8", QUANT, match, **changes)


@pytest.mark.parametrize("changes,match", [
    (dict(rows=-1), "rows=-1"), (dict(k=0), "k=0"), (dict(dtype=3), "dtype 3"),
    (dict(eps=-1.0), "eps -1"), (dict(eps=float("nan")), "eps"), (dict(ldq=8), "ldq=8"),
    (dict(ldx=8), "ldx=8"), (dict(residual=P, ldr=8), "ldr=8"), (dict(out=P, ldo=8), "ldo=8"),
    (dict(dev=99), "bad device 99"), (dict(w=None), "null buffer"), (dict(x=None), "null buffer"),
    (dict(x=P + 1), "misaligned"), (dict(residual=P + 1, ldr=64), "misaligned"),
    (dict(residual=P, ldr=64, out=P, ldo=72), "needs its row stride"),
    (dict(out=P, ldo=72), "needs its row stride"),
])
def test_rms_norm_refusals(changes, match):
    refused("futon_cuda_rms_norm_f8", NORM, match, **changes)


@pytest.mark.parametrize("changes,match", [
    (dict(m=-1), "m=-1"), (dict(n=0), "n=0"), (dict(k=0), "k=0"), (dict(dst_dtype=3), "output dtype 3"),
    (dict(lda=63), "lda=63"), (dict(ldb=48), "ldb=48"), (dict(ldd=7), "ldd=7"),
    (dict(lda=72), "not multiples of 16"), (dict(ldb=72), "not multiples of 16"),
    (dict(lda=1 << 40), "row strides"), (dict(dev=-2), "bad device -2"),
    (dict(dst=None), "null buffer"), (dict(a_scales=None), "null buffer"),
    (dict(b_scales=None), "null buffer"), (dict(a=P + 8), "start at multiples of 16"),
    (dict(b=P + 1), "start at multiples of 16"), (dict(dst=P + 2), "misaligned"),
    (dict(bias=P + 1), "misaligned"),
    (dict(m=2 ** 31 - 2048, n=2 ** 31 - 2048, ldd=2 ** 31), "too many tiles"),
    (dict(m=2 ** 31 - 1), "m=2147483647"),
])
def test_matmul_refusals(changes, match):
    refused("futon_cuda_matmul_t_f8", MATMUL, match, **changes)


@pytest.mark.parametrize("changes,match", [
    (dict(groups=0), "groups=0"), (dict(groups=1025), "groups=1025"), (dict(dtype=0), "operand dtype 0"),
    (dict(dtype=4), "operand dtype 4"), (dict(dtype=3), "null buffer"), (dict(offsets=None), "null buffer"),
    (dict(n=2 ** 30, ldd=2 ** 30), "rows"), (dict(lda=68), "not multiples of 16"),
    (dict(offsets=P + 2), "misaligned"),
])
def test_grouped_refusals(changes, match):
    refused("futon_cuda_matmul_t_grouped", GROUPED, match, **changes)


def test_no_rows_is_a_no_op():
    for fn, base, change in (("futon_cuda_quantize_f8", QUANT, dict(rows=0, q=None, src=None)),
                             ("futon_cuda_rms_norm_f8", NORM, dict(rows=0, x=None)),
                             ("futon_cuda_matmul_t_f8", MATMUL, dict(m=0, dst=None, a=None)),
                             ("futon_cuda_matmul_t_grouped", GROUPED, dict(m=0, offsets=None))):
        _lib.call(fn, *dict(base, **change).values())


def test_messages_fit_short_buffers():
    """A caller's short or missing message buffer is respected."""
    args = list(dict(QUANT, k=0).values())
    fn = _lib.lib().futon_cuda_quantize_f8
    buf = C.create_string_buffer(b"x" * 16, 16)
    assert fn(*args, buf, 8) == E
    assert len(buf.value) == 7 and buf.raw[8:] == b"x" * 8
    assert fn(*args, None, 0) == E


# ---- the tensor layer ----

torch = pytest.importorskip("torch")
F8 = torch.float8_e4m3fn


def codes(r, k):
    return torch.zeros(r, k, dtype=torch.uint8).view(F8)


def raises(match, fn, *a, **k):
    with pytest.raises(FutonError, match=match) as ei:
        fn(*a, **k)
    assert ei.value.code == E


def test_tensors_on_the_host_are_refused():
    x = torch.zeros(2, 64)
    raises("CUDA device", f8.quantize_f8, x)
    raises("CUDA device", f8.rms_norm_f8, x, torch.ones(64), 1e-6)
    s = torch.zeros(2, 1)
    raises("CUDA device", f8.matmul_t_f8, codes(2, 64), s, codes(8, 64), torch.zeros(1, 1))
    raises("CUDA device", f8.matmul_t_grouped, torch.zeros(2, 64, dtype=torch.float16),
           torch.zeros(3, 8, 64, dtype=torch.float16), torch.zeros(4, dtype=torch.int32))


def test_quantize_tensor_checks():
    x = torch.zeros(4, 64)
    raises("activation 'relu'", f8.quantize_f8, x, activation="relu")
    raises("block_rows=2", f8.quantize_f8, x, block_rows=2)
    raises("float64", f8.quantize_f8, x.double())
    raises("3 dimensions", f8.quantize_f8, x.view(2, 2, 64))
    raises("contiguous", f8.quantize_f8, torch.zeros(64, 4).t())
    raises("rows overlap", f8.quantize_f8, x[:1].expand(4, 64))
    raises(r"\[fc1 \| gate\]", f8.quantize_f8, x[:, :63], activation="swiglu")
    raises("k=0", f8.quantize_f8, x[:, :0])
    raises("codes must be", f8.quantize_f8, x, out=(codes(4, 32), torch.zeros(4, 1)))
    raises("codes must be", f8.quantize_f8, x, out=(torch.zeros(4, 64), torch.zeros(4, 1)))
    raises("scales must be", f8.quantize_f8, x, out=(codes(4, 64), torch.zeros(4, 2)))


def test_norm_tensor_checks():
    x, w = torch.zeros(4, 64), torch.ones(64)
    raises("weight must be", f8.rms_norm_f8, x, w.half(), 1e-6)
    raises("weight must be", f8.rms_norm_f8, x, w[:32], 1e-6)
    raises("residual must be", f8.rms_norm_f8, x, w, 1e-6, residual=x.half())
    raises("residual_out must be", f8.rms_norm_f8, x, w, 1e-6, residual=x, residual_out=x[:2])
    raises("int32", f8.rms_norm_f8, x.int(), w, 1e-6)


def test_product_tensor_checks():
    a, sa, b, sb = codes(4, 64), torch.zeros(4, 1), codes(8, 64), torch.zeros(1, 1)
    raises("float8_e4m3fn", f8.matmul_t_f8, a.float(), sa, b, sb)
    raises("shapes", f8.matmul_t_f8, a, sa, codes(8, 32), sb)
    raises("a_scales must be", f8.matmul_t_f8, a, torch.zeros(1, 4), b, sb)
    raises("b_scales must be", f8.matmul_t_f8, a, sa, b, torch.zeros(8, 1))
    raises("bias must be", f8.matmul_t_f8, a, sa, b, sb, bias=torch.zeros(4))
    raises("out must have shape", f8.matmul_t_f8, a, sa, b, sb, out=torch.zeros(8, 4))
    raises("out must be float32", f8.matmul_t_f8, a, sa, b, sb, out=torch.zeros(4, 8).double())
    raises("out_dtype", f8.matmul_t_f8, a, sa, b, sb, out=torch.zeros(4, 8), out_dtype=torch.float16)


def test_grouped_tensor_checks():
    h = torch.float16
    a, b, off = torch.zeros(4, 64, dtype=h), torch.zeros(2, 8, 64, dtype=h), torch.zeros(3, dtype=torch.int32)
    raises("differ", f8.matmul_t_grouped, a, b.bfloat16(), off)
    raises("takes float8_e4m3fn", f8.matmul_t_grouped, a.float(), b.float(), off)
    raises("offsets must be", f8.matmul_t_grouped, a, b, off.long())
    raises("offsets must be", f8.matmul_t_grouped, a, b, off[:2])
    raises("take no scales", f8.matmul_t_grouped, a, b, off, a_scales=torch.zeros(4, 1))
    raises("need a_scales", f8.matmul_t_grouped, codes(4, 64), codes(16, 64).view(2, 8, 64), off)
    raises("elements apart", f8.matmul_t_grouped, a, torch.zeros(2, 16, 64, dtype=h)[:, :8], off)
    raises("bias must be", f8.matmul_t_grouped, a, b, off, bias=torch.zeros(8))


def test_gradients_are_refused():
    """No backward pass: a tensor that records gradients is refused, and
    passes that check where gradients are off."""
    x = torch.zeros(2, 64, requires_grad=True)
    w = torch.ones(64, requires_grad=True)
    raises("no backward pass", f8.quantize_f8, x)
    raises("no backward pass", f8.rms_norm_f8, x.detach(), w, 1e-6)
    with torch.no_grad():
        raises("CUDA device", f8.quantize_f8, x)


def test_wrong_kinds_of_argument():
    x = torch.zeros(2, 64)
    raises("src must be a tensor, got list", f8.quantize_f8, [1.0])
    raises("weight must be a tensor", f8.rms_norm_f8, x, None, 1e-6)
    raises("pair", f8.quantize_f8, x, out=x)
    raises("torch.dtype", f8.matmul_t_f8, codes(2, 64), torch.zeros(2, 1), codes(8, 64),
           torch.zeros(1, 1), out_dtype="float32")
    with pytest.raises(TypeError):
        f8.rms_norm_f8(x, torch.ones(64), "eps")
