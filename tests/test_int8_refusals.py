"""What the operators on 8-bit integers refuse, on the CPU: C entries by their status codes before any
launch, argument checks, derivatives."""

import ctypes
import os

import pytest
import torch
from torch.autograd import forward_ad

from tests import int8_util as I


@pytest.fixture(scope="module")
def lib():
    from torchtitan_amd import _lib

    if not os.path.exists(_lib.library_path()):
        from torchtitan_amd import build

        build.build()
    return _lib.lib()


@pytest.fixture(scope="module")
def at():
    """A 16-byte aligned address (nothing is read: every call here ends before a launch)."""
    buf = ctypes.create_string_buffer(80)
    yield (ctypes.addressof(buf) + 15) // 16 * 16


def test_rows(lib, at):
    quant = lambda ld=64, rows=4, cols=64, dtype=0, x=at, q=at, s=at: lib.moe_int8_quant_rows(x, ld, rows, cols, dtype, q, s, None)  # noqa: E731
    dequant = lambda rows=4, cols=64, dtype=0, q=at, s=at, x=at: lib.moe_int8_dequant_rows(q, s, rows, cols, dtype, x, None)  # noqa: E731
    assert quant(rows=0, x=None, q=None, s=None) == 0 and dequant(rows=0, x=None, q=None, s=None) == 0
    for bad in (dict(rows=-1), dict(cols=0), dict(dtype=2), dict(dtype=-1), dict(x=None), dict(q=None), dict(s=None)):
        assert quant(**bad) == -1 and dequant(**bad) == -1, bad
    assert quant(ld=63) == -1
    assert quant(rows=2 ** 31) == -2 and dequant(rows=2 ** 31) == -2


def test_rows_past_the_columns_that_are_counted(lib, at):
    """Columns are counted in 32 bits, with steps past the last one."""
    big = 2 ** 30 + 8
    assert lib.moe_int8_quant_rows(at, big, 1, big, 0, at, at, None) == -2
    assert lib.moe_int8_dequant_rows(at, at, 1, big, 0, at, None) == -2


def test_sizes_that_an_entry_would_cut(monkeypatch):
    """Sizes past 32 bits are refused before they reach an entry, which would take their low part."""
    from torchtitan_amd import ops

    monkeypatch.setattr(ops, "_int8_device", lambda *a: 0)
    monkeypatch.setattr(ops, "_int8_launch", lambda *a: pytest.fail("launched"))
    x = torch.zeros(1, dtype=torch.bfloat16)
    for cols in (2 ** 30 + 1, 2 ** 32 + 16):
        with pytest.raises(ValueError, match="columns"):
            ops._int8_quantize(x.expand(1, cols))
        with pytest.raises(ValueError, match="columns"):
            ops._int8_dequantize(torch.zeros(1, dtype=torch.int8).expand(cols), torch.zeros(()), torch.bfloat16)
    for n in (2 ** 22 + 1, 2 ** 32 + 8):
        with pytest.raises(ValueError, match="output channels"):
            ops._linear_int8(x.expand(1, 16), torch.zeros(1, dtype=torch.int8).expand(n, 16), torch.zeros(1).expand(n))


def test_linear(lib, at):
    def run(r=4, e=2, k=64, n=32, x=at, w=at, s=at, b=None, bd=0, c=at, ws=at, size=1 << 40, y=at, dtype=0):
        return lib.moe_int8_linear(x, dtype, w, s, b, bd, c, r, e, k, n, ws, size, y, None)

    assert run(r=0, x=None, w=None) == 0
    for bad, want in ((dict(r=-1), -1), (dict(e=0), -1), (dict(e=1025), -1), (dict(k=0), -1), (dict(n=0), -1), (dict(k=72), -2),
                      (dict(k=131088), -2), (dict(n=(1 << 22) + 1), -2), (dict(r=2 ** 30), -2), (dict(r=2 ** 27, n=2 ** 12), -2),
                      (dict(dtype=2), -1), (dict(bd=2), -1), (dict(c=None), -1), (dict(x=None), -1), (dict(w=None), -1),
                      (dict(s=None), -1), (dict(y=None), -1), (dict(x=at + 2), -1), (dict(w=at + 8), -1), (dict(y=at + 4), -1),
                      (dict(r=400000, ws=None), -1), (dict(r=400000, ws=at + 8), -1), (dict(r=400000, size=400000 * 128), -4)):
        assert run(**bad) == want, bad
    ws = lib.moe_int8_linear_workspace_bytes
    assert ws(-1, 2, 64, 64) == -1 and ws(4, 0, 64, 64) == -1 and ws(4, 2, 72, 64) == -2 and ws(4, 2, 64, 0) == -1
    assert ws(1, 1, 64, 64) == 0  # few rows are quantized on the way
    assert ws(4000, 2, 2880, 2880) == 4000 * 2944 + 16128  # codes of whole stages of 128, and scales


def test_layers(lib, at):
    def silu(r=4, e=2, d=64, h=32, x=at, w=at, c=at, ws=at, size=1 << 40, y=at):
        return lib.moe_int8_swiglu(x, w, at, at, at, w, at, c, r, e, d, h, ws, size, y, None)

    def oss(r=4, e=2, d=64, h=32, b1=at, b2=at, bd=0, size=1 << 40, m=at):
        return lib.moe_int8_oss(at, m, at, b1, at, at, b2, bd, at, r, e, d, h, 7.0, at, size, at, None)

    assert silu(r=0) == 0 and oss(r=0) == 0
    for bad, want in ((dict(r=-1), -1), (dict(e=0), -1), (dict(e=1025), -1), (dict(d=0), -1), (dict(h=0), -1), (dict(d=72), -2),
                      (dict(h=40), -2), (dict(d=131088), -2), (dict(h=2 ** 30), -2), (dict(r=2 ** 30), -2), (dict(size=64), -4)):
        assert silu(**bad) == want and oss(**bad) == want, bad
    for bad in (dict(c=None), dict(x=None), dict(w=None), dict(ws=None), dict(y=None), dict(x=at + 2), dict(w=at + 8), dict(ws=at + 8),
                dict(y=at + 8)):
        assert silu(**bad) == -1, bad
    for bad in (dict(b1=None), dict(b2=None), dict(bd=2), dict(m=None)):
        assert oss(**bad) == -1, bad
    ws = lib.moe_int8_layer_workspace_bytes
    assert ws(-1, 2, 64, 64) == -1 and ws(4, 0, 64, 64) == -1 and ws(4, 2, 72, 64) == -1 and ws(4, 2, 64, 72) == -1
    assert ws(0, 2, 64, 64) == 0 and ws(1000, 2, 272, 144) == 1000 * 4 * 144 + 1000 * 384 + 4096


def _w(*shape):
    return torch.zeros(*shape, dtype=torch.int8), torch.ones(*shape[:-1])


def test_arguments(monkeypatch):
    from torchtitan_amd import ops

    monkeypatch.setattr(ops, "_int8_device", lambda op, *t: 0)
    bf = torch.bfloat16
    x, w, ws, c = torch.zeros(4, 64, dtype=bf), _w(32, 64), _w(2, 32, 64), torch.tensor([2, 2])
    for call, what in (
            (lambda: ops.int8_quantize(x.half()), "bfloat16 and float32"),
            (lambda: ops.int8_dequantize(*w, torch.float16), "bfloat16 and float32"),
            (lambda: ops.int8_dequantize(w[0].float(), w[1]), "int8"),
            (lambda: ops.int8_dequantize(w[0], w[1].double()), "float32 scales"),
            (lambda: ops.linear_int8(x.half(), *w), "bfloat16 and float32"),
            (lambda: ops.linear_int8(x, w[0].view(torch.uint8), w[1]), "int8"),
            (lambda: ops.linear_int8(x, *w, torch.zeros(32).half()), "biases"),
            (lambda: ops.grouped_linear_int8(x, *ws, c.float()), "integer counts"),
            (lambda: ops.grouped_linear_int8(x, *ws, c > 1), "integer counts"),
            (lambda: ops.swiglu_ffn_int8(x.float(), *w, *_w(64, 32), *w), "bfloat16 x"),
            (lambda: ops.grouped_swiglu_int8(x.float(), *ws, *_w(2, 64, 32), *ws, c), "bfloat16 x"),
            (lambda: ops.grouped_swiglu_oss_int8(x, *ws, torch.zeros(2, 32, dtype=bf), *_w(2, 64, 16), torch.zeros(2, 64), c, 7.0), "one dtype")):
        with pytest.raises(TypeError, match=what):
            call()
    b16 = torch.zeros(2, 32, dtype=bf)
    for call in (lambda: ops.int8_quantize(x[0, 0]), lambda: ops.int8_quantize(x[:, :0]), lambda: ops.int8_dequantize(w[0], w[1][1:]),
                 lambda: ops.int8_dequantize(w[0][:, :0], w[1]), lambda: ops.int8_dequantize(w[0], w[1][0]),
                 lambda: ops.linear_int8(x[:, :48], *w), lambda: ops.linear_int8(x, *ws), lambda: ops.linear_int8(x[0, 0], *w),
                 lambda: ops.linear_int8(x, *w, torch.zeros(31)), lambda: ops.linear_int8(x[:, :40], *_w(32, 40)),
                 lambda: ops.linear_int8(x[:, :0], *_w(32, 0)), lambda: ops.linear_int8(x, *_w(0, 64)),
                 lambda: ops.linear_int8(x[:, :1].expand(4, 131088), *_w(1, 131088)),
                 lambda: ops.grouped_linear_int8(x, *w, c), lambda: ops.grouped_linear_int8(x[0], *ws, c),
                 lambda: ops.grouped_linear_int8(x, *ws, c[:1]), lambda: ops.grouped_linear_int8(x, *ws, c.view(1, 2)),
                 lambda: ops.grouped_linear_int8(x, *ws, c, torch.zeros(32)), lambda: ops.grouped_linear_int8(x, *_w(0, 32, 64), c[:0]),
                 lambda: ops.grouped_linear_int8(x, *_w(1025, 1, 64), torch.zeros(1025, dtype=torch.int64)),
                 lambda: ops.swiglu_ffn_int8(x, *w, *w, *w), lambda: ops.swiglu_ffn_int8(x, *w, *_w(64, 32), *_w(31, 64)),
                 lambda: ops.swiglu_ffn_int8(x, *_w(24, 64), *_w(64, 24), *_w(24, 64)),
                 lambda: ops.swiglu_ffn_int8(x, *ws, *_w(2, 64, 32), *ws),
                 lambda: ops.grouped_swiglu_int8(x, *ws, *_w(2, 32, 64), *ws, c), lambda: ops.grouped_swiglu_int8(x, *w, *_w(64, 32), *w, c),
                 lambda: ops.grouped_swiglu_int8(x, *ws, *_w(2, 64, 32), *ws, c[:1]),
                 lambda: ops.grouped_swiglu_oss_int8(x, *ws, b16, *_w(2, 64, 16), x[:2], c, -1.0),
                 lambda: ops.grouped_swiglu_oss_int8(x, *ws, b16, *_w(2, 64, 16), x[:2], c, float("nan")),
                 lambda: ops.grouped_swiglu_oss_int8(x, *ws, b16[:, 1:], *_w(2, 64, 16), x[:2], c, 7.0),
                 lambda: ops.grouped_swiglu_oss_int8(x, *ws, b16, *_w(2, 64, 32), x[:2], c, 7.0),
                 lambda: ops.grouped_swiglu_oss_int8(x, *_w(2, 33, 64), b16, *_w(2, 64, 16), x[:2], c, 7.0)):
        with pytest.raises(ValueError):
            call()


def test_ops_refuse_cpu_tensors():
    from torchtitan_amd import _lib, ops

    for _, f, x in _calls(ops):
        with torch.no_grad(), pytest.raises(_lib.MoEKernelError, match="GPU"):
            f(x)
    for call in (lambda: ops.int8_quantize(torch.ones(2, 4)), lambda: ops.int8_dequantize(*_w(2, 4))):
        with pytest.raises(_lib.MoEKernelError, match="GPU"):
            call()


def _calls(ns):
    """(operator, a call of it by one of its differentiable inputs, that input)."""
    bf = torch.bfloat16
    x, c, w, w2 = torch.ones(4, 64, dtype=bf), torch.tensor([2, 2]), _w(32, 64), _w(64, 32)
    ws, w2s, m2 = _w(2, 32, 64), _w(2, 64, 32), _w(2, 64, 16)
    b, bs, b2 = torch.ones(32), torch.ones(2, 32), torch.ones(2, 64)
    for name, args in (("linear_int8", [x, *w, b]), ("grouped_linear_int8", [x, *ws, c, bs]), ("swiglu_ffn_int8", [x, *w, *w2, *w]),
                       ("grouped_swiglu_int8", [x, *ws, *w2s, *ws, c]), ("grouped_swiglu_oss_int8", [x, *ws, bs, *m2, b2, c, 7.0])):
        for i, t in enumerate(args):
            if isinstance(t, torch.Tensor) and t.is_floating_point():
                yield name, lambda v, i=i, name=name, args=args: getattr(ns, name)(*args[:i], v, *args[i + 1:]), t


def _dual(f, x):
    with forward_ad.dual_level():
        f(forward_ad.make_dual(x, torch.ones_like(x)))


@pytest.mark.parametrize("derive", [
    lambda f, x: f(x.clone().requires_grad_(True)), _dual, lambda f, x: torch.func.jvp(f, (x,), (torch.ones_like(x),)),
    lambda f, x: torch.func.grad(lambda t: f(t).float().sum())(x)])
def test_derivatives(derive):
    """Those of activations, scales and biases are refused, not dropped, through the package and
    through the dispatcher."""
    from torchtitan_amd import _lib, ops

    for ns in (ops, torch.ops.moe_mi355x_int8):
        for name, f, x in _calls(ns):
            with pytest.raises(RuntimeError, match="no gradients"):
                derive(f, x)
            with torch.no_grad(), pytest.raises(_lib.MoEKernelError, match="GPU"):  # nothing to lose
                f(x.clone().requires_grad_(True))


def test_fake():
    """Shapes and types without data, on every operator."""
    from torch._subclasses.fake_tensor import FakeTensorMode

    from torchtitan_amd import ops

    with FakeTensorMode():
        x, c = torch.empty(2, 3, 64, dtype=torch.bfloat16, device="cuda"), torch.empty(2, dtype=torch.int64, device="cuda")
        w = lambda *s: (torch.empty(*s, dtype=torch.int8, device="cuda"), torch.empty(*s[:-1], device="cuda"))  # noqa: E731
        q, s = ops.int8_quantize(x)
        assert q.dtype == torch.int8 and q.shape == x.shape and s.dtype == torch.float32 and s.shape == (2, 3)
        assert ops.int8_dequantize(q, s, torch.float32).dtype == torch.float32
        y = ops.linear_int8(x, *w(5, 64))
        assert y.shape == (2, 3, 5) and y.dtype == x.dtype
        assert ops.grouped_linear_int8(x[0], *w(2, 5, 64), c).shape == (3, 5)
        assert ops.swiglu_ffn_int8(x, *w(32, 64), *w(64, 32), *w(32, 64)).shape == x.shape
        assert ops.grouped_swiglu_int8(x[0], *w(2, 32, 64), *w(2, 64, 32), *w(2, 32, 64), c).shape == (3, 64)
        assert ops.grouped_swiglu_oss_int8(x[0], *w(2, 64, 64), torch.empty(2, 64, device="cuda"), *w(2, 64, 32),
                                           torch.empty(2, 64, device="cuda"), c, 7.0).shape == (3, 64)


def test_oracle():
    """The 64-bit form that the GPU tests compare with: hand-worked rows, and that a code is the nearest
    integer to its value over the scale."""
    q, s = I.pack(torch.tensor([[127.0, 0.5, 1.5, -2.5, 63.49], [2.0, 1.0, -1.0, 0.0, 0.0079], [0.0] * 5]))
    assert q.tolist() == [[127, 0, 2, -2, 63], [127, 64, -64, 0, 1], [0] * 5]
    assert s.tolist() == [1.0, torch.tensor(2 / 127).item(), 2.0 ** -126]
    x = torch.randn(40, 300, generator=torch.Generator().manual_seed(1))
    q, s = I.pack(x)
    assert q.abs().max() == 127 and bool((q.abs().amax(-1) == 127).all())
    assert bool(((x.double() - I.values(q, s)).abs() <= s.double().unsqueeze(-1) * (0.5 + 127 * 2.0 ** -23)).all())
    y, tol = I.linear(x, q, s, None, torch.float32)
    assert torch.equal(y, y.T) and bool((tol < 2.0 ** -21 * y.abs() + 2.0 ** -130).all())
