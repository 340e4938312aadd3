"""Models whose dense linears run on the 8-bit integer path (weights and activations), against the fp32 oracle, and the
engine's bitwise properties on it."""
import pytest
import torch

pytestmark = pytest.mark.gpu

RECIPE = "all,mlp:int8,attn:int8,gdn:int8"


def _build(moe=False, recipe=RECIPE):
    from velogb10_b200.checkpoint.synthetic import SyntheticSource
    from velogb10_b200.config import tiny_hybrid, tiny_moe
    from velogb10_b200.models.weights import ModelBuilder
    cfg = tiny_moe() if moe else tiny_hybrid()
    return cfg, ModelBuilder(cfg, SyntheticSource(cfg, 0, "cuda", std=0.05), recipe=recipe, device="cuda").build()


def _prompt(cfg, n, seed=1):
    return torch.randint(0, cfg.vocab_size, (n,), generator=torch.Generator().manual_seed(seed)).tolist()


# Rounding an input to 8 bits adds noise of step / sqrt(12) with step = max / 127: 0.75 % of a 256-wide Gaussian row, about
# 2 % of a SwiGLU row (largest value 8 times the rms). The branches' errors add like the branches themselves, so logits made
# from the same weight codes and unquantised activations differ by about 2 %: 6 % is three times that.
NOISE = 0.06


def test_prefill_and_decode_match_oracle():
    from velogb10_b200.models.oracle import OracleModel
    from velogb10_b200.models.runtime import GpuModel
    from velogb10_b200.ops import lib
    cfg, w = _build()
    orc = OracleModel(_build()[1])
    gm = GpuModel(w, keep_canonical=True)
    assert {q.fmt for _, q in w.linears()} >= {"int8", "nvfp4"}
    gm.alloc_state(2, 2 + 17, 256)
    orc.alloc_state(2, 2 + 17, 256)
    prompt = _prompt(cfg, 40)
    lg, _ = gm.prefill(1, prompt)
    lo, _ = orc.prefill(1, prompt)
    assert ((lg.float().cpu() - lo).norm() / lo.norm()).item() < NOISE
    tok = int(lo.argmax())
    for i in range(3):
        lgd, _ = gm.decode([tok], [40 + i], [1])
        lod, _ = orc.decode([tok], [40 + i], [1])
        assert ((lgd[0].float().cpu() - lod[0]).norm() / lod[0].norm()).item() < NOISE
        tok = int(lod[0].argmax())
    lib.check_err_word()


def test_moe_with_int8_mixers_and_shared_expert():
    """Expert selection is a step function of the router logits, so noise in them changes outputs without bound: the
    reference (the same codes decoded to bf16) lends its router logits to the int8 run."""
    from velogb10_b200.models.runtime import GpuModel
    from velogb10_b200.ops import lib
    cfg, w = _build(moe=True)
    ref = _build(moe=True)[1]
    for _, q in ref.linears():
        if q.fmt == "int8":
            q.w, q.fmt, q.codes, q.row_scale = q.dequant(torch.bfloat16), "bf16", None, None
    a, b = GpuModel(w, keep_canonical=True), GpuModel(ref, keep_canonical=True)
    for m in (a, b):
        m.alloc_state(2, 2 + 17, 256)
    seen = []
    b.router_logits_hook = lambda logits, n: seen.append(logits[:n].clone())
    a.router_logits_hook = lambda logits, n: logits[:n].copy_(seen.pop(0))
    prompt = _prompt(cfg, 40)
    want = b.prefill(1, prompt)[0].clone()
    got = a.prefill(1, prompt)[0]
    assert ((got.float() - want.float()).norm() / want.float().norm()).item() < NOISE
    for i, tok in enumerate((3, 77, 500)):
        want = b.decode([tok], [40 + i], [1])[0].clone()
        got = a.decode([tok], [40 + i], [1])[0]
        assert ((got.float() - want.float()).norm() / want.float().norm()).item() < NOISE
    assert not seen
    lib.check_err_word()


def test_batch_verify_and_graph_are_bitwise_sequential():
    from velogb10_b200.models.runtime import GpuModel
    cfg, w = _build()
    gm = GpuModel(w, keep_canonical=True)
    gm.alloc_state(4, 4 + 17, 512)
    prompts = [_prompt(cfg, n, n) for n in (16, 23, 70, 33)]
    firsts = [int(gm.prefill(s, p)[0].argmax()) for s, p in enumerate(prompts)]
    keep = [t.clone() for t in (gm.S, gm.conv, gm.kc, gm.vc)]

    def restore():
        for t, k in zip((gm.S, gm.conv, gm.kc, gm.vc), keep):
            t.copy_(k)

    pos = [len(p) for p in prompts]
    batch = gm.decode(firsts, pos, [0, 1, 2, 3])[0].clone()
    restore()
    for s in range(4):
        assert torch.equal(gm.decode([firsts[s]], [pos[s]], [s])[0][0], batch[s]), s
    restore()
    toks = [firsts[2], 5, 7, 11]
    verify = gm.verify(2, toks, pos[2], ckpt_base=4)[0].clone()
    restore()
    for t in range(4):
        assert torch.equal(gm.decode([toks[t]], [pos[2] + t], [2])[0][0], verify[t]), t
    restore()
    gm.capture_decode(4)
    restore()
    gm.replay_decode(firsts, pos, [0, 1, 2, 3])
    torch.cuda.synchronize()
    assert gm.ws.out_tok[:4].tolist() == batch.argmax(-1).tolist()


def test_gates_cover_int8_linears(capsys):
    """The batch-invariance gate and the GEMM probe name the formats they ran; an int8 linear that broke must fail the gate."""
    import json
    from velogb10_b200 import gates
    from velogb10_b200.models.runtime import GpuModel
    cfg, w = _build()
    gm = GpuModel(w, keep_canonical=True)
    int8 = [q for _, q in w.linears() if q.fmt == "int8"]
    assert gates.gate_binv(gm, cfg) == 0
    out = json.loads(capsys.readouterr().out.strip().splitlines()[-1])
    assert out["formats"]["int8"] == min(12, len(int8)) and out["formats"]["nvfp4"] > 0 and out["rel_l2"] < 1e-3, out
    assert gates.probe_gemm(gm, cfg) == 0
    rows = json.loads(capsys.readouterr().out.strip().splitlines()[-1])["rows"]
    assert {r["format"] for r in rows} >= {"int8", "nvfp4"} and all(r["us"] > 0 and r["GBs"] > 0 for r in rows)
    scale = int8[0].row_scale
    int8[0].row_scale = scale * torch.where(torch.arange(scale.numel(), device=scale.device) % 2 == 0, 1.0, 1.1)
    deq = int8[0].dequant
    int8[0].dequant = lambda dtype=torch.bfloat16: (int8[0].codes.float() * scale[:, None]).to(dtype)     # plain reference kept
    assert gates.gate_binv(gm, cfg) == 1
    int8[0].dequant = deq


def test_no_f16_rows_beside_int8_rows(monkeypatch):
    """A dense layer's norms and SwiGLU hand int8 rows to their only reader: no f16 copy is written, no buffer for one is held.
    The range probe reads the copy, so it gets one, with the same logits."""
    from velogb10_b200.models import runtime
    cfg, w = _build()
    asked, norm = [], runtime.I8.add_rmsnorm_int8
    monkeypatch.setattr(runtime.I8, "add_rmsnorm_int8", lambda *a, **k: asked.append(k.get("out16")) or norm(*a, **k))
    gm = runtime.GpuModel(w, keep_canonical=True)
    gm.alloc_state(2, 2 + 17, 256)
    prompt = _prompt(cfg, 40)
    want = gm.prefill(1, prompt)[0].clone()
    gm.decode([3], [40], [1])
    assert len(asked) == 4 * cfg.num_layers and all(o is None for o in asked)
    kept = {L.attn.o.k if L.attn is not None else L.gdn.out.k for L in w.layers}          # mixer outputs are f16
    assert set(gm.ws._a16) | set(gm.ws_prefill._a16) == kept
    gm.zero_slot(1)
    gm.cap_debug, asked[:] = True, []
    assert torch.equal(gm.prefill(1, prompt)[0], want)
    assert all(o is not None for o in asked)
