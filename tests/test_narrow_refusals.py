"""What the MXFP4 operators and the 8-bit activations refuse, on the CPU: C entries by their
status codes before any launch, argument checks, converters and packed modules."""

import ctypes
from types import SimpleNamespace

import pytest
import torch

from tests import narrow_util as N

DIMS = SimpleNamespace(pp_enabled=False, cp_enabled=False, ep_enabled=False)


@pytest.fixture(scope="module")
def lib():
    import os

    from torchtitan_amd import _lib

    if not os.path.exists(_lib.library_path()):
        from torchtitan_amd import build

        build.build()
    return _lib.lib()


def _aligned(n=64):
    buf = ctypes.create_string_buffer(n + 16)
    return buf, (ctypes.addressof(buf) + 15) // 16 * 16


def test_quantizers(lib):
    null = None
    keep, at = _aligned()
    for fn, args in ((lib.moe_mxfp4_quant_rows, (null, 4, 64, 64, 0, null, null, null)),
                     (lib.moe_mxfp4_dequant_rows, (null, null, 4, 64, 64, 0, null, null))):
        assert fn(*args) == -1  # null tensors
    quant = lib.moe_mxfp4_quant_rows
    assert quant(null, 0, 64, 64, 0, null, null, null) == 0
    for rows, cols, q_cols, dtype in ((-1, 64, 64, 0), (4, 0, 0, 0), (4, 48, 64, 0), (4, 64, 32, 0), (4, 64, 80, 0), (4, 64, 64, 2)):
        assert quant(at, rows, cols, q_cols, dtype, at, at, null) == -1
    assert quant(at + 2, 4, 64, 64, 0, at, at, null) == -1  # misaligned
    assert quant(at, 4, 64, 64, 0, at + 4, at, null) == -1
    assert lib.moe_mxfp4_padded_cols(32) == 256 and lib.moe_mxfp4_padded_cols(256) == 256
    assert lib.moe_mxfp4_padded_cols(288) == 512 and lib.moe_mxfp4_padded_cols(48) == -1
    assert lib.moe_keep8_rows(null, 0, 64, null, null, null) == 0
    for rows, cols in ((-1, 64), (2, 40), (2, 0)):
        assert lib.moe_keep8_rows(at, rows, cols, at, at, null) == -1
        assert lib.moe_restore8_rows(at, at, rows, cols, at, null) == -1
    assert lib.moe_keep8_rows(null, 2, 64, at, at, null) == -1
    assert lib.moe_restore8_rows(at, null, 2, 64, at, null) == -1


def test_products(lib):
    null = None
    keep, at = _aligned()
    fwd = lambda r, e, d, h, ws_bytes=1 << 40, x=at, w=at, ws=at: lib.moe_mxfp4_swiglu_fwd(  # noqa: E731
        x, w, w, w, w, w, w, at, r, e, d, h, ws, ws_bytes, at, null)
    assert fwd(0, 2, 64, 64) == 0
    for r, e, d, h, want in ((-1, 2, 64, 64, -1), (4, 0, 64, 64, -1), (4, 1025, 64, 64, -1), (4, 2, 0, 64, -1),
                             (4, 2, 80, 64, -2), (4, 2, 64, 48, -2), (2 ** 30, 2, 64, 64, -2), (4, 2, 2 ** 23, 64, -2)):
        assert fwd(r, e, d, h) == want
    assert fwd(4, 2, 64, 64, ws_bytes=16) == -4
    for bad in (dict(x=null), dict(w=null), dict(ws=null), dict(x=at + 2), dict(w=at + 8), dict(ws=at + 1)):
        assert fwd(4, 2, 64, 64, **bad) == -1
    assert lib.moe_mxfp4_swiglu_fwd(at, at, at, at, at, at, at, null, 4, 2, 64, 64, at, 1 << 40, at, null) == -1
    oss = lambda b1, b2: lib.moe_mxfp4_oss_fwd(at, at, at, b1, at, at, b2, at, 4, 2, 64, 64, 7.0, at, 1 << 40, at, null)  # noqa: E731
    assert oss(null, at) == -1 and oss(at, null) == -1
    # the workspace: rows of x and h padded to 256 columns, and odd scale rows for the wide kernel
    ws = lib.moe_mxfp4_workspace_bytes
    assert ws(0, 2, 64, 64) == 0 and ws(-1, 2, 64, 64) == -1 and ws(4, 2, 48, 64) == -1
    assert ws(2, 4, 64, 64) == 2 * (2 * 128 + 256)
    assert ws(1000, 4, 96, 64) == 2 * (128000 + 8192)
    assert ws(2000, 4, 96, 64) == 2 * (256000 + 16128) + 4 * 2 * 64 * 8
    # the training products take even numbers of blocks
    gate = lambda r, d, h, q=at: lib.moe_mxfp4_gemm_gate_up_keep(q, at, at, at, at, at, at, r, 2, d, h, at, at, at, at, at, at, null)  # noqa: E731
    down = lambda r, d, h, q=at: lib.moe_mxfp4_gemm_down(q, at, at, at, at, r, 2, d, h, at, null)  # noqa: E731
    assert gate(4, 96, 64) == -2 and down(4, 64, 96) == -2
    assert gate(4, 64, 64, null) == -1 and down(4, 64, 64, null) == -1
    assert gate(0, 64, 64, null) == 0 and down(0, 64, 64, null) == 0
    assert lib.moe_grouped_gemm_gate_up_keep8(null, null, null, at, 4, 2, 64, 64, null, null, null, null, null, null) == -1
    assert lib.moe_grouped_gemm_gate_up_keep8(null, null, null, at, 0, 2, 64, 64, null, null, null, null, null, null) == 0
    assert lib.moe_grouped_gemm_gate_up_keep8(at, at, at, at, 4, 2, 64, 64, at, null, null, null, at, null) == -1
    assert lib.moe_grouped_gemm_bwd_dgu_keep8(at, at, null, at, at, at, at, 4, 2, 64, 64, at, null, null) == -1
    for bad in ((at + 8, at, at, at), (at, at + 1, at, at), (at, at, at + 4, at), (at, at, at, at + 1)):  # read in wide pieces
        assert lib.moe_grouped_gemm_bwd_dgu_keep8(at, at, *bad, at, 4, 2, 64, 64, at, null, null) == -1
    assert lib.moe_grouped_gemm_bwd_dx_once(null, at, at, at, 4, 2, 64, 64, at, null) == -1


def test_packed_arguments():
    from torchtitan_amd import ops

    q, s = torch.zeros(3, 5, 32, dtype=torch.uint8), torch.zeros(3, 5, 2, dtype=torch.uint8)
    ops._check_packed("op", "w", q, s, (3, 5, 64))
    for a, b in ((q.float(), s), (q, s.int())):
        with pytest.raises(TypeError, match="uint8"):
            ops._check_packed("op", "w", a, b)
    for a, b in ((q, s[:, :4]), (q, s[0]), (q, torch.zeros(3, 5, 3, dtype=torch.uint8)), (q[..., :24], s),
                 (q[..., :0], s[..., :0])):
        with pytest.raises(ValueError):
            ops._check_packed("op", "w", a, b)
    with pytest.raises(ValueError, match="expects w"):
        ops._check_packed("op", "w", q, s, (3, 4, 64))


def test_kept_arguments():
    from torchtitan_amd import ops

    assert ops._carve((1, 256, 257, 0, 5)) == ((0, 256, 512, 1024, 1024), 1280)
    offsets, size = ops._ckpt8_layout(3, 64, 128)
    assert offsets == (0, 256, 512, 1024, 1280, 1792) and size == 2048
    offsets, size = ops._mxfp4_train_layout(3, 2, 64, 128)  # w of 16384 elements, rows of 256 columns, g and u of 128
    assert offsets == (0, 8192, 8704, 16896, 17408, 25600, 26112, 26624, 26880, 27392, 27648, 28160, 28416, 28928)
    assert size == 29184
    dy, kept = torch.zeros(3, 64), torch.zeros(2048, dtype=torch.uint8)
    wide = torch.zeros(4096, dtype=torch.uint8)[::2]
    assert ops._check_kept("op", kept, 2048, dy) is kept and ops._check_kept("op", wide, 2048, dy).is_contiguous()
    with pytest.raises(TypeError, match="uint8"):
        ops._check_kept("op", kept.view(torch.int8), 2048, dy)
    for bad in (kept[1:], kept.view(2, -1)):
        with pytest.raises(ValueError, match="2048 bytes"):
            ops._check_kept("op", bad, 2048, dy)


def test_expert_arguments(monkeypatch):
    from torchtitan_amd import ops

    monkeypatch.setattr(ops, "require_gpu", lambda *t: None)
    bf = torch.bfloat16
    x, w1, w2 = torch.zeros(4, 64, dtype=bf), torch.zeros(2, 128, 64, dtype=bf), torch.zeros(2, 64, 128, dtype=bf)
    c = torch.tensor([2, 2])
    ops._check_experts("op", x, w1, w2, w1, c, 64)
    with pytest.raises(TypeError, match="bfloat16 w1"):
        ops._check_experts("op", x, w1.float(), w2, w1, c, 64)
    with pytest.raises(TypeError, match="integer counts"):
        ops._check_experts("op", x, w1, w2, w1, c.float(), 64)
    for args in ((x[0], w1, w2, w1, c), (x, w1[0], w2, w1, c), (x, w1, w1, w1, c), (x, w1, w2, w2, c),
                 (x[:, :32], w1, w2, w1, c), (x, w1, w2, w1, c[:1]), (x, w1, w2, w1, c.view(1, 2))):
        with pytest.raises(ValueError):
            ops._check_experts("op", *args, 64)
    with pytest.raises(ValueError, match="multiples of 64"):
        ops._check_experts("op", x[:, :32], w1[..., :32].contiguous(), w2[:, :32], w1[..., :32].contiguous(), c, 64)
    with pytest.raises(ValueError, match="1 to 1024 experts"):
        ops._check_dims("op", 1025, 64, 64, 32)
    with pytest.raises(TypeError, match="bfloat16 x"):
        ops._check_mxfp4_rows("op", x.float(), torch.zeros(2, 128, 32, dtype=torch.uint8), c)
    with pytest.raises(ValueError):
        ops._check_mxfp4_rows("op", x, torch.zeros(2, 127, 32, dtype=torch.uint8), c, 2)
    with pytest.raises(TypeError, match="bfloat16 and float32"):
        ops._mx_dtype("op", torch.float16)
    with pytest.raises(ValueError, match="whole blocks of 32"):
        ops._check_mx_matrix("op", 48)


def test_ops_refuse_cpu_tensors():
    from torchtitan_amd import _lib, ops

    bf = torch.bfloat16
    x, w, c = torch.zeros(4, 64, dtype=bf), torch.zeros(1, 64, 64, dtype=bf), torch.tensor([4])
    q, s = torch.zeros(1, 64, 32, dtype=torch.uint8), torch.zeros(1, 64, 2, dtype=torch.uint8)
    for call in (lambda: ops.mxfp4_quantize(x), lambda: ops.mxfp4_dequantize(q, s),
                 lambda: ops.grouped_swiglu_mxfp4(x, q, s, q, s, q, s, c),
                 lambda: ops.grouped_swiglu_oss_mxfp4(x, q, s, x, q, s, x, c, 7.0),
                 lambda: ops.grouped_swiglu_ckpt8(x, w, w, w, c), lambda: ops.grouped_swiglu_mxfp4_train(x, w, w, w, c)):
        with pytest.raises(_lib.MoEKernelError, match="GPU"):
            call()


def _experts():
    from torchtitan_amd import GroupedExperts

    return GroupedExperts.Config(dim=64, hidden_dim=64, num_experts=2).build()


def test_recipes_exclude_each_other():
    from torchtitan_amd import quantization as Q

    for first, second in (("mxfp4", "ckpt8"), ("ckpt8", "mxfp8"), ("float8", "mxfp4"), ("mxfp8", "ckpt8")):
        model = torch.nn.ModuleDict({"a": torch.nn.ModuleDict({"experts": _experts()}), "other": _experts()})
        assert Q._mark_experts(model, ["a.experts"], first) == ["a.experts"]
        with pytest.raises(ValueError, match="already converted"):
            Q._mark_experts(model, ["experts", "other"], second)
        assert not getattr(model["other"], second)  # nothing is marked half way
        assert Q._mark_experts(model, ["a.experts"], first) == ["a.experts"]
    model = torch.nn.ModuleDict({"experts": _experts()})
    Q._mark_experts(model, ["experts"], "float8")
    Q._mark_experts(model, ["experts"], "mxfp8")  # as before


def test_converters_need_the_hardware(monkeypatch):
    from torchtitan_amd import quantization as Q

    monkeypatch.setattr(Q, "has_gfx950", lambda: False)
    for cls in (Q.MXFP4Converter, Q.MXFP8ActivationCheckpointConverter, Q.MXFP4WeightConverter):
        with pytest.raises(ValueError, match="gfx950"):
            cls.Config(fqns=["experts"]).build(parallel_dims=DIMS, model_compile_enabled=False)
    monkeypatch.setattr(Q, "has_gfx950", lambda: True)
    for cls, attr in ((Q.MXFP4Converter, "mxfp4"), (Q.MXFP8ActivationCheckpointConverter, "ckpt8")):
        model = torch.nn.ModuleDict({"experts": _experts(), "rest": _experts()})
        conv = cls.Config(fqns="experts,").build(parallel_dims=DIMS, model_compile_enabled=False)
        assert conv.convert(model) == ["experts"]
        assert getattr(model["experts"], attr) and not getattr(model["rest"], attr)
    assert Q.find_pad_multiple([Q.MXFP4Converter.Config()]) is None


def test_packed_modules(monkeypatch):
    """Buffers and their shapes; a checkpoint's blocks go in as they are; what does not fit is refused."""
    from torchtitan_amd import ops
    from torchtitan_amd.mxfp4 import MXFP4GptOssGroupedExperts, MXFP4GroupedExperts
    from torchtitan_amd.quantization import MXFP4WeightConverter

    m = MXFP4GptOssGroupedExperts.Config(dim=64, hidden_dim=96, num_experts=2, swiglu_limit=5.0).build()
    assert {k: tuple(v.shape) for k, v in m.state_dict().items()} == {
        "mlp1_weight_blocks": (2, 192, 32), "mlp1_weight_scales": (2, 192, 2), "mlp2_weight_blocks": (2, 64, 48),
        "mlp2_weight_scales": (2, 64, 3), "mlp1_bias": (2, 192), "mlp2_bias": (2, 64)}
    assert not list(m.parameters()) and m.swiglu_limit == 5.0
    at = "model.layers.3.mlp.experts."
    gen = torch.Generator().manual_seed(0)
    u8 = lambda *s: torch.randint(0, 256, s, generator=gen, dtype=torch.uint8)  # noqa: E731
    hf = {at + "gate_up_proj_blocks": u8(2, 192, 2, 16), at + "gate_up_proj_scales": u8(2, 192, 2),
          at + "gate_up_proj_bias": torch.randn(2, 192), at + "down_proj_blocks": u8(2, 64, 3, 16),
          at + "down_proj_scales": u8(2, 64, 3), at + "down_proj_bias": torch.randn(2, 64)}
    m.load_hf(hf, 3)
    assert torch.equal(m.mlp1_weight_blocks.view(2, 192, 2, 16), hf[at + "gate_up_proj_blocks"])
    assert torch.equal(m.mlp2_weight_scales, hf[at + "down_proj_scales"])
    assert torch.equal(m.mlp2_bias, hf[at + "down_proj_bias"].bfloat16())
    for key, bad in (("gate_up_proj_blocks", u8(2, 190, 2, 16)), ("down_proj_scales", u8(2, 64, 2)),
                     ("down_proj_blocks", u8(2, 64, 3, 16).float()), ("gate_up_proj_bias", torch.randn(2, 96))):
        with pytest.raises(ValueError):
            m.load_hf({**hf, at + key: bad}, 3)
    with pytest.raises(ValueError, match="whole blocks"):
        MXFP4GroupedExperts.Config(dim=48, hidden_dim=64, num_experts=2).build()
    # the converter replaces experts by packed ones (the packing itself on the CPU here)
    monkeypatch.setattr(ops, "mxfp4_quantize", N.pack4)
    monkeypatch.setattr("torchtitan_amd.quantization.has_gfx950", lambda: True)
    model = torch.nn.ModuleDict({"layer": torch.nn.ModuleDict({"experts": _experts()}), "rest": _experts()})
    weights = {}
    for n, p in model["layer"]["experts"].named_parameters():
        weights[n] = torch.nn.init.normal_(p).detach().clone()
    conv = MXFP4WeightConverter.Config(fqns=["layer"]).build(parallel_dims=DIMS, model_compile_enabled=False)
    assert conv.convert(model) == ["layer.experts"]
    packed = model["layer"]["experts"]
    assert type(packed) is MXFP4GroupedExperts and packed.num_experts == 2
    for n, w in weights.items():
        assert torch.equal(N.unpack4(*packed.packed(n)), N.q4(w))
    with pytest.raises(ValueError, match="does not fit"):
        packed.pack("w1", torch.zeros(2, 32, 64))


def test_oracle_formats():
    """The 64-bit formats that the GPU tests compare with: hand-worked values and the nearest-value
    property on random blocks."""
    v = torch.zeros(1, 32)
    v[0, :8] = torch.tensor([6.0, 5.0, -3.5, 2.5, 1.75, 0.75, 0.25, -0.2501])
    assert N.q4(v)[0, :8].tolist() == [6.0, 4.0, -4.0, 2.0, 2.0, 1.0, 0.0, -0.5]
    assert N.q4(v * 1.0001)[0, 0] == 6.0 and N.pack4(v * 1.0001)[1].item() == 128
    assert N.pack4(v)[1].item() == 127 and N.pack4(v * 0)[1].item() == 0
    x = torch.randn(50, 32, generator=torch.Generator().manual_seed(1), dtype=torch.float64)
    s = torch.exp2(N.pack4(x)[1].double() - 127)  # [50, 1]
    grid = torch.cat([N.E2M1, -N.E2M1]) * s  # [50, 16]
    near = (x.unsqueeze(-1) - grid.unsqueeze(1)).abs().amin(-1)
    assert torch.equal((N.q4(x) - x).abs(), near)
    assert bool((x.abs().amax(-1) <= 6 * s.squeeze(-1)).all()) and bool((x.abs().amax(-1) > 3 * s.squeeze(-1)).all())
    got8 = N.q8(x)
    assert torch.equal((got8 / N._scale(x.abs().amax(-1, keepdim=True), 448.0)).float().to(torch.float8_e4m3fn).double(),
                       got8 / N._scale(x.abs().amax(-1, keepdim=True), 448.0))
    assert bool(((got8 - x).abs() <= 2.0 ** -4 * x.abs() + 2.0 ** -10 * N._scale(x.abs().amax(-1, keepdim=True), 448.0)).all())
