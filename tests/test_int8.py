"""The 8-bit integer path on the host: weight codec, containers, and the refusals of the wrappers (all of them before
anything is enqueued)."""
import pytest
import torch

from velogb10_b200.models.weights import QLinear, fuse_rows
from velogb10_b200.ops import int8 as I8
from velogb10_b200.ops.lib import KernelError
from velogb10_b200.quant import codec


@pytest.mark.parametrize("m,k", [(1, 1), (5, 16), (64, 33), (200, 515)])
def test_codec_is_within_half_a_step(m, k):
    g = torch.Generator().manual_seed(m * 1000 + k)
    w = torch.randn(m, k, generator=g)
    q = codec.quantize_int8(w)
    assert q.codes.dtype == torch.int8 and q.codes.shape == (m, k)
    assert q.codes.data_ptr() % 16 == 0 and (m == 1 or q.codes.stride(0) % 16 == 0)
    assert torch.equal(q.row_scale, w.abs().amax(-1) / 127.0)
    assert (q.codes.abs().amax(-1) == 127).all()
    # half a step, plus the roundings of the division (2^-24 of at most 127 steps) and of the scale
    off = (q.codes.double() * q.row_scale.double()[:, None] - w.double()).abs() / q.row_scale.double()[:, None]
    assert off.max() <= 0.5 + 127 * 2 * 2.0 ** -24
    assert torch.equal(codec.dequantize_int8(q.codes, q.row_scale, torch.float32), q.codes.float() * q.row_scale[:, None])


def test_zero_rows_and_fake_quant():
    w = torch.zeros(3, 20)
    w[1] = torch.arange(20.0) - 10
    q = codec.quantize_int8(w)
    assert (q.codes[0] == 0).all() and (q.codes[2] == 0).all() and float(q.row_scale[0]) == 2.0 ** -120
    assert (codec.fake_quant(w, "int8") - w).abs().max() <= 10 / 127 / 2 * 1.0001
    assert codec.bits_per_weight("int8", 32) == 9.0


def test_container_keeps_rows_on_16_byte_boundaries():
    g = torch.Generator().manual_seed(0)
    w = torch.randn(24, 50, generator=g)
    q = QLinear.from_dense(w, "int8")
    assert q.fmt == "int8" and q.codes.stride(0) == 64 and torch.equal(q.dequant(), q.codes.float() * q.row_scale[:, None])
    two = fuse_rows([q, q])
    assert two.m == 48 and torch.equal(two.codes[24:], q.codes) and two.codes.stride(0) % 16 == 0
    part = q.rows(3, 9)
    assert torch.equal(part.codes, q.codes[3:9]) and part.codes.stride(0) % 16 == 0 and torch.equal(part.row_scale, q.row_scale[3:9])
    cut = q.cols(16, 48)
    assert torch.equal(cut.codes, q.codes[:, 16:48]) and cut.codes.stride(0) % 16 == 0
    assert q.to("cpu").codes.stride(0) % 16 == 0
    mixed = fuse_rows([q, QLinear.from_dense(w, "fp8")])
    assert mixed.fmt == "bf16"


def test_recipe_and_checkpoint(tmp_path):
    from velogb10_b200.checkpoint import io
    from velogb10_b200.checkpoint.synthetic import SyntheticSource, synthetic_state_dict
    from velogb10_b200.config import tiny_hybrid
    from velogb10_b200.models.weights import ModelBuilder
    from velogb10_b200.quant.recipe import parse_recipe
    recipe = "all,mlp:int8,attn:int8,gdn:int8"
    assert parse_recipe(recipe)["mlp"] == "int8" and parse_recipe(recipe)["lmhead"] == "nvfp4"
    assert "mlp" not in parse_recipe("mlp:int8,-mlp:int8")
    for bad in ("all:int8", "lmhead:int8", "expert:int8", "embed:int8", "router:int8", "mtp:int8"):
        with pytest.raises(ValueError, match="int8 is for"):
            parse_recipe(bad)
    cfg = tiny_hybrid(False)
    out = str(tmp_path / "ck")
    stats = io.write_checkpoint(out, synthetic_state_dict(cfg, seed=0).items(), cfg.to_hf_dict(), recipe)
    assert stats["int8"] > 0 and stats["nvfp4"] > 0
    direct = ModelBuilder(cfg, SyntheticSource(cfg, 0), recipe=recipe).build()
    loaded = ModelBuilder(cfg, io.SafetensorsSource(out)).build()
    n = 0
    for (name, a), (name2, b) in zip(direct.linears(), loaded.linears()):
        assert name == name2 and a.fmt == b.fmt
        if a.fmt == "int8":
            n += 1
            assert torch.equal(a.codes, b.codes) and torch.equal(a.row_scale, b.row_scale)
            assert b.codes.stride(0) % 16 == 0 and b.codes.data_ptr() % 16 == 0
    assert n == 2 * cfg.num_layers + 2 * cfg.num_layers          # mixer in / out and MLP in / down of every layer


def test_int8_tensors_without_int8_kernels_load_as_bf16():
    from velogb10_b200.config import tiny_hybrid
    from velogb10_b200.models.weights import ModelBuilder
    g = torch.Generator().manual_seed(0)
    two, three = torch.randn(32, 48, generator=g), torch.randn(4, 16, 32, generator=g)
    a, b = codec.quantize_int8(two), codec.quantize_int8(three.reshape(64, 32))
    tensors = {"lm_head.weight": a.codes, "lm_head.weight_scale": a.row_scale,
               "layers.0.mlp.experts.gate_up_proj": b.codes.reshape(4, 16, 32),
               "layers.0.mlp.experts.gate_up_proj.weight_scale": b.row_scale.reshape(4, 16),
               "layers.0.mlp.up_proj.weight": a.codes, "layers.0.mlp.up_proj.weight_scale": a.row_scale[:, None]}

    class Source:
        def get(self, name):
            return tensors.get(name)

    mb = ModelBuilder(tiny_hybrid(False), Source())
    head, experts, up = mb.linear("lm_head"), mb.linear("layers.0.mlp.experts.gate_up_proj", ""), mb.linear("layers.0.mlp.up_proj")
    assert head.fmt == "bf16" and torch.equal(head.w, codec.dequantize_int8(a.codes, a.row_scale))
    assert experts.fmt == "bf16" and experts.experts == 4 and torch.equal(experts.w, codec.dequantize_int8(b.codes, b.row_scale))
    assert up.fmt == "int8" and torch.equal(up.codes, a.codes) and torch.equal(up.row_scale, a.row_scale)


def test_other_linears_refuse_int8_weights():
    from velogb10_b200.ops import gemm as G
    q = _w(16, 32)
    with pytest.raises(KernelError, match="int8"):
        G.prepare(q)
    with pytest.raises(KernelError, match="int8"):
        G.linear_simt(q, torch.zeros(1, 32, dtype=torch.float16))


def _act(n, k):
    return I8.Int8Act(codec.rows16(torch.zeros((n, k), dtype=torch.int8)), torch.ones(n))


def _w(m, k):
    return QLinear("int8", m, k, codes=codec.rows16(torch.zeros((m, k), dtype=torch.int8)), row_scale=torch.ones(m))


BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.mark.parametrize("what,call", [
    ("expected a matrix", lambda: I8.quantize_act_int8(torch.zeros(8))),
    ("not supported", lambda: I8.quantize_act_int8(torch.zeros(2, 8, dtype=torch.float64))),
    ("rows asked for", lambda: I8.quantize_act_int8(torch.zeros(2, 8), n=3)),
    ("rows asked for", lambda: I8.quantize_act_int8(torch.zeros(2, 8), n=-1)),
    ("contiguous", lambda: I8.quantize_act_int8(torch.zeros(8, 2).t())),
    ("contiguous", lambda: I8.quantize_act_int8(torch.zeros(1, 8).expand(2, 8))),
    ("outside", lambda: I8.quantize_act_int8(torch.zeros(2, 0))),
    ("outside", lambda: I8.quantize_act_int8(torch.zeros(1, I8.MAX_K + 1))),
    ("out.q", lambda: I8.quantize_act_int8(torch.zeros(2, 8), out=_act(1, 8))),
    ("out.q", lambda: I8.quantize_act_int8(torch.zeros(2, 8), out=_act(2, 9))),
    ("out.scale", lambda: I8.quantize_act_int8(torch.zeros(2, 8), out=I8.Int8Act(_act(2, 8).q, torch.ones(1)))),
    ("out.scale", lambda: I8.quantize_act_int8(torch.zeros(2, 8), out=I8.Int8Act(_act(2, 8).q, torch.ones(2, dtype=F16)))),
    ("gu", lambda: I8.swiglu_int8(torch.zeros(2, 7, dtype=BF))),
    ("gu", lambda: I8.swiglu_int8(torch.zeros(2, 8, dtype=BF), inter=3)),
    ("gu", lambda: I8.swiglu_int8(torch.zeros(2, 8))),
    ("eps", lambda: I8.add_rmsnorm_int8(torch.zeros(2, 8, dtype=BF), None, torch.ones(8), 0.0)),
    ("eps", lambda: I8.add_rmsnorm_int8(torch.zeros(2, 8, dtype=BF), None, torch.ones(8), float("nan"))),
    ("w:", lambda: I8.add_rmsnorm_int8(torch.zeros(2, 8, dtype=BF), None, torch.ones(9), 1e-6)),
    ("w:", lambda: I8.add_rmsnorm_int8(torch.zeros(2, 8, dtype=BF), None, torch.ones(8, dtype=BF), 1e-6)),
    ("w:", lambda: I8.add_rmsnorm_int8(torch.zeros(2, 8, dtype=BF), None, torch.ones(16)[::2], 1e-6)),
    ("res", lambda: I8.add_rmsnorm_int8(torch.zeros(2, 8), None, torch.ones(8), 1e-6)),
    ("delta", lambda: I8.add_rmsnorm_int8(torch.zeros(2, 8, dtype=BF), torch.zeros(1, 8, dtype=BF), torch.ones(8), 1e-6)),
    ("delta", lambda: I8.add_rmsnorm_int8(torch.zeros(2, 8, dtype=BF), torch.zeros(2, 8), torch.ones(8), 1e-6)),
    ("out16", lambda: I8.add_rmsnorm_int8(torch.zeros(2, 8, dtype=BF), None, torch.ones(8), 1e-6, out16=torch.zeros(2, 9, dtype=F16))),
    ("act.q", lambda: I8.dequantize_act_int8(I8.Int8Act(torch.zeros(2, 8), torch.ones(2)))),
    ("act.scale", lambda: I8.dequantize_act_int8(I8.Int8Act(_act(2, 8).q, torch.ones(1)))),
    ("dtype", lambda: I8.dequantize_act_int8(_act(2, 8), dtype=torch.float64)),
    ("out", lambda: I8.dequantize_act_int8(_act(2, 8), out=torch.zeros(2, 9))),
    ("takes int8 weights", lambda: I8.linear_int8(QLinear.from_dense(torch.zeros(4, 16), "fp8"), _act(2, 16))),
    ("act.q", lambda: I8.linear_int8(_w(4, 32), _act(2, 16))),
    ("rows asked for", lambda: I8.linear_int8(_w(4, 32), _act(2, 32), n=3)),
    ("16-byte", lambda: I8.linear_int8(_w(4, 33), I8.Int8Act(torch.zeros((2, 33), dtype=torch.int8), torch.ones(2)))),
    ("16-byte", lambda: I8.linear_int8(_w(4, 32), I8.Int8Act(torch.zeros(80, dtype=torch.int8)[1:65].view(2, 32), torch.ones(2)))),
    ("16-byte", lambda: I8.linear_int8(QLinear("int8", 2, 33, codes=torch.zeros((2, 33), dtype=torch.int8), row_scale=torch.ones(2)), _act(2, 33))),
    ("row_scale", lambda: I8.linear_int8(QLinear("int8", 4, 32, codes=_w(4, 32).codes, row_scale=torch.ones(3)), _act(2, 32))),
    ("codes", lambda: I8.linear_int8(QLinear("int8", 5, 32, codes=_w(4, 32).codes, row_scale=torch.ones(5)), _act(2, 32))),
    ("act.scale", lambda: I8.linear_int8(_w(4, 32), I8.Int8Act(_act(2, 32).q, torch.ones(1)))),
    ("K must be", lambda: I8.linear_int8(_w(1, I8.MAX_K + 1), _act(1, I8.MAX_K + 1))),
    ("out", lambda: I8.linear_int8(_w(4, 32), _act(2, 32), out=torch.zeros(2, 5))),
    ("out", lambda: I8.linear_int8(_w(4, 32), _act(2, 32), out=torch.zeros(2, 4, dtype=F16))),
    ("out", lambda: I8.linear_int8(_w(4, 32), _act(2, 32), out=torch.zeros(4, 2).t())),
    ("CUDA", lambda: I8.linear_int8(_w(4, 32), _act(2, 32))),
    ("CUDA", lambda: I8.quantize_act_int8(torch.zeros(2, 8))),
    ("CUDA", lambda: I8.swiglu_int8(torch.zeros(2, 8, dtype=BF))),
    ("CUDA", lambda: I8.add_rmsnorm_int8(torch.zeros(2, 8, dtype=BF), None, torch.ones(8), 1e-6)),
    ("CUDA", lambda: I8.dequantize_act_int8(_act(2, 8))),
])
def test_refusals(what, call):
    with pytest.raises(KernelError, match=what):
        call()


def test_codec_rounds_exact_halves_to_even():
    """bf16 rows hold exact halves (127 w / max = n + 1/2), which a quotient of rounded numbers puts on either side. The rule
    is checked in whole numbers: every bf16 value here is an integer times 2^-20."""
    g = torch.Generator().manual_seed(7)
    w = (torch.randn(40, 4001, generator=g) * 0.9).clamp(-7, 7).bfloat16()
    w = torch.where(w.abs() < 2.0 ** -12, torch.zeros_like(w), w)
    q = codec.quantize_int8(w)
    v = (w.double() * 2 ** 20).long()
    assert torch.equal(v.double() * 2.0 ** -20, w.double())
    amax = v.abs().amax(-1, keepdim=True)
    twice, rem = (254 * v.abs()) // amax, (254 * v.abs()) % amax           # quotient in half steps
    half = (twice % 2 == 1) & (rem == 0)
    want = torch.where(half, (twice // 2 + 1) // 2 * 2, (twice + 1) // 2) * v.sign()
    assert half.sum() > 20
    assert torch.equal(q.codes.long(), want)
    assert torch.equal(q.row_scale, (amax.squeeze(-1).double() * 2.0 ** -20 / 127).float())


def test_norm_behind_a_pending_reduction_quantises_the_residual(monkeypatch):
    """Tensor-parallel decode widths leave a sum to the norm kernel, longer inputs do not. The int8 rows come from the fp32 norm
    of the residual in both cases, not from the f16 copy."""
    from types import SimpleNamespace
    from velogb10_b200.models import runtime
    calls = []
    monkeypatch.setattr(runtime.G, "add_rmsnorm_fp4_ar", lambda *a, **k: calls.append("sum") or ("bq", "sfb", "g0"))
    monkeypatch.setattr(runtime.I8, "add_rmsnorm_int8", lambda res, delta, w, eps, n, **k: calls.append((res, delta, n, k["out"])) or k["out"])
    gm = object.__new__(runtime.GpuModel)
    gm.cfg, gm.comm, gm.use_fp4 = SimpleNamespace(rms_eps=1e-6), None, True
    x, out = torch.zeros(16, 32, dtype=BF), _act(16, 32)
    ws = SimpleNamespace(x=x, xn16=torch.zeros(16, 32, dtype=F16), delta=torch.zeros_like(x), i8=lambda width, tag="": out)
    for mode in (1, 2):
        gm._pending_ar, calls[:] = mode, []
        assert gm._norm(ws, ws.delta, torch.zeros(32), 3, _w(8, 32)) is out
        assert calls[0] == "sum" and calls[1][0] is x and calls[1][1] is None and calls[1][2] == 3 and gm._pending_ar == 0
    gm._pending_ar = 1
    assert gm._norm(ws, ws.delta, torch.zeros(32), 3, QLinear("nvfp4", 16, 32)) == ("bq", "sfb", "g0")


def _builder(tensors):
    from velogb10_b200.config import tiny_hybrid
    from velogb10_b200.models.weights import DictSource, ModelBuilder
    return ModelBuilder(tiny_hybrid(False), DictSource(tensors))


def test_checkpoint_scales_and_zero_points():
    """What stands beside int8 codes decides what they mean: other layouts than a scale a row are refused at load."""
    g = torch.Generator().manual_seed(0)
    a = codec.quantize_int8(torch.randn(32, 48, generator=g))
    name = "layers.0.mlp.up_proj"
    base = {name + ".weight": a.codes, name + ".weight_scale": a.row_scale[:, None]}
    zeros = torch.zeros(32, 1, dtype=torch.int8)
    q = _builder({**base, name + ".weight_zero_point": zeros}).linear(name)
    assert torch.equal(q.codes, a.codes) and torch.equal(q.row_scale, a.row_scale)
    one = _builder({**base, name + ".weight_scale": torch.tensor([0.5]).bfloat16()}).linear(name)
    assert one.row_scale.shape == (32,) and one.row_scale.is_contiguous() and (one.row_scale == 0.5).all()
    assert torch.equal(one.dequant(), a.codes.float() * 0.5)
    for extra, what in (({name + ".weight_zero_point": zeros + 1}, "zero point"),
                        ({name + ".weight_scale": torch.ones(32, 3)}, "96 scales for 32"),
                        ({name + ".weight_scale": torch.ones(31)}, "31 scales for 32")):
        with pytest.raises(ValueError, match=what):
            _builder({**base, **extra}).linear(name)
    with pytest.raises(ValueError, match="without a weight_scale"):
        _builder({name + ".weight": a.codes}).linear(name)
    head = {"lm_head.weight": a.codes, "lm_head.weight_scale": a.row_scale}          # decoded to bf16: the same rules
    with pytest.raises(ValueError, match="zero point"):
        _builder({**head, "lm_head.weight_zero_point": zeros + 1}).linear("lm_head")
    assert torch.equal(_builder({**head, "lm_head.weight_scale": torch.tensor(2.0)}).linear("lm_head").w, (a.codes.float() * 2).bfloat16())


def test_requant_re_encodes_int8_gdn_projections(tmp_path):
    """``gdn4`` means GDN projections in NVFP4, whatever 8-bit format they came in; the int8 MLP stays as it is."""
    from velogb10_b200.checkpoint import io
    from velogb10_b200.checkpoint.synthetic import synthetic_state_dict
    from velogb10_b200.config import tiny_hybrid
    from velogb10_b200.models.weights import ModelBuilder
    cfg = tiny_hybrid(False)
    a, b = str(tmp_path / "a"), str(tmp_path / "b")
    io.write_checkpoint(a, synthetic_state_dict(cfg, seed=0).items(), cfg.to_hf_dict(), "all,mlp:int8,gdn:int8")
    stats = io.requant_gdn(a, b)
    before = dict(ModelBuilder(cfg, io.SafetensorsSource(a)).build().linears())
    after = dict(ModelBuilder(cfg, io.SafetensorsSource(b)).build().linears())
    gdn = [n for n in before if n.endswith(("in_proj", "gdn.out")) or ".gdn" in n]
    assert stats["requant"] > 0 and gdn and all(before[n].fmt == "int8" and after[n].fmt == "nvfp4" for n in gdn)
    for n in before:
        if n not in gdn:
            assert before[n].fmt == after[n].fmt
            if before[n].fmt == "int8":
                assert torch.equal(before[n].codes, after[n].codes) and torch.equal(before[n].row_scale, after[n].row_scale)


def test_checkpoint_names_its_layout(tmp_path):
    import json
    from velogb10_b200.checkpoint import io
    from velogb10_b200.checkpoint.synthetic import synthetic_state_dict
    from velogb10_b200.config import tiny_hybrid
    cfg = tiny_hybrid(False)

    def label(d):
        return json.load(open(d + "/config.json"))["quantization_config"]["format"]

    for i, (recipe, want, after) in enumerate((("all", "nvfp4-pack-quantized", "nvfp4-pack-quantized"),
                                               ("all,gdn:fp8", "nvfp4-pack-quantized", "nvfp4-pack-quantized"),
                                               ("all,gdn:int8", "mixed-precision", "nvfp4-pack-quantized"),
                                               ("all,mlp:int8,gdn:int8", "mixed-precision", "mixed-precision"),
                                               ("mlp:int8,attn:int8,gdn:int8", "int-quantized", "mixed-precision"))):
        a, b = str(tmp_path / f"a{i}"), str(tmp_path / f"b{i}")
        io.write_checkpoint(a, synthetic_state_dict(cfg, seed=0).items(), cfg.to_hf_dict(), recipe)
        assert label(a) == want
        io.requant_gdn(a, b)
        assert label(b) == after


_WITHOUT = """
import torch
for holder, name in ((torch._C, "_cuda_getDevice"), (torch._C, "_cuda_getCurrentRawStream"),
                     (torch._C._dynamo.guards, "_empty_strided_cuda")):
    if hasattr(holder, name):
        delattr(holder, name)
import velogb10_b200.engine.device_sampler, velogb10_b200.models.runtime, velogb10_b200.parallel.comm
from velogb10_b200.ops import int8, lib
assert lib._raw_stream is None and lib._empty_strided_cuda is None and lib.current_index is torch.cuda.current_device
t = lib.empty_beside(torch.zeros(2), (3, 5), (16, 1), torch.int8)
assert t.shape == (3, 5) and t.stride() == (16, 1) and t.dtype == torch.int8
print("imported")
"""


def test_imports_without_pytorchs_private_calls():
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", _WITHOUT], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "imported" in r.stdout, r.stderr[-2000:]


@pytest.mark.parametrize("eps", [1e-46, 2.0 ** -127, 2.0 ** -101, 1e39, float("inf"), -1e-6])
def test_eps_outside_fp32(eps):
    """An eps that fp32 does not hold: zero rows would become NaN, or all rows zero."""
    with pytest.raises(KernelError, match="eps"):
        I8.add_rmsnorm_int8(torch.zeros(2, 8, dtype=BF), None, torch.ones(8), eps)
