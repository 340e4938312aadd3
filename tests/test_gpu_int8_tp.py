"""int8 models sharded over ranks. One GPU plays both ranks: each rank's model runs in a host thread of its own, one at a time, and
hands over where a collective would run, so no kernel ever waits for another rank."""
import threading

import pytest
import torch

pytestmark = pytest.mark.gpu

NOISE = 0.06           # three times the noise of 8-bit activations in the logits, as for the unsharded models
RECIPE = "all,mlp:int8,attn:int8,gdn:int8"


class _Ranks:
    def __init__(self, world):
        self.world, self.turn = world, threading.Lock()
        self.barrier = threading.Barrier(world, timeout=120)
        self.boxes = [[None] * world, [None] * world]
        self.comms = [_Comm(self, r) for r in range(world)]

    def run(self, fn):
        """``fn(rank)`` on every rank; the results in rank order."""
        out, errors = [None] * self.world, []

        def body(rank):
            try:
                with self.turn:
                    out[rank] = fn(rank)
            except BaseException as e:  # noqa: BLE001
                errors.append(e)
                self.barrier.abort()

        threads = [threading.Thread(target=body, args=(r,)) for r in range(self.world)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        if errors:
            raise errors[0]
        return out


class _Comm:
    """What the runtime asks of a communicator on its plain path (collectives as calls of their own)."""
    use_nccl, use_mm, mc = True, False, 0

    def __init__(self, ranks, rank):
        self.ranks, self.rank, self.world, self.step = ranks, rank, ranks.world, 0

    def _exchange(self, t):
        box = self.ranks.boxes[self.step & 1]             # the other box may still be read by a rank one step behind
        self.step += 1
        box[self.rank] = t.clone()
        self.ranks.turn.release()
        try:
            self.ranks.barrier.wait()
        finally:
            self.ranks.turn.acquire()
        return list(box)

    def all_reduce_rows(self, t, n):
        parts = self._exchange(t[:n])
        t[:n].copy_(sum(p.float() for p in parts))

    def gather_logits(self, t):
        return torch.cat(self._exchange(t), -1)


def _cfg(moe):
    from velogb10_b200.config import tiny_hybrid, tiny_moe
    cfg = (tiny_moe if moe else tiny_hybrid)(mtp=False)
    cfg.num_heads, cfg.num_kv_heads, cfg.lin_num_k_heads, cfg.lin_num_v_heads = 4, 2, 4, 8
    return cfg


def _weights(cfg, rank=0, world=1, recipe=RECIPE):
    from velogb10_b200.checkpoint.synthetic import SyntheticSource
    from velogb10_b200.models.weights import ModelBuilder
    return ModelBuilder(cfg, SyntheticSource(cfg, 0, "cuda", std=0.05), recipe=recipe, device="cuda", tp_rank=rank, tp_world=world).build()


def _as_bf16(w):
    """The same codes decoded: what the model computes without 8-bit activations."""
    for _, q in w.linears():
        if q.fmt == "int8":
            q.w, q.fmt, q.codes, q.row_scale = q.dequant(torch.bfloat16), "bf16", None, None
    return w


def _rel(a, b):
    return ((a.float() - b.float()).norm() / b.float().norm()).item()


def test_two_ranks_dense():
    """Sharded prefill and decode against the unsharded model without 8-bit activations; ranks agree bit for bit; verify and
    batched decode have the bits of single-token decode."""
    from velogb10_b200.models.runtime import GpuModel
    from velogb10_b200.ops import lib
    cfg, ranks = _cfg(False), _Ranks(2)
    ref = GpuModel(_as_bf16(_weights(cfg)), keep_canonical=True)
    tp = [GpuModel(_weights(cfg, r, 2), comm=ranks.comms[r]) for r in range(2)]
    whole = dict(_weights(cfg).linears())
    for r, m in enumerate(tp):
        shards = dict(m.w.linears())
        assert {q.fmt for q in shards.values()} >= {"int8", "nvfp4"}
        assert shards["layers.0.mlp.gate_up"].m * 2 == whole["layers.0.mlp.gate_up"].m
        assert shards["layers.0.mlp.down"].k * 2 == whole["layers.0.mlp.down"].k
    for m in [ref] + tp:
        m.alloc_state(3, 3 + 17, 512)
    g = torch.Generator().manual_seed(5)
    prompt = torch.randint(0, cfg.vocab_size, (90,), generator=g).tolist()
    want = ref.prefill(0, prompt)[0].clone()
    got = ranks.run(lambda r: tp[r].prefill(0, prompt)[0].clone())
    assert torch.equal(got[0], got[1]) and torch.equal(tp[0].ws_prefill.x, tp[1].ws_prefill.x)
    assert got[0].shape == want.shape and _rel(got[0], want) < NOISE
    toks = [int(want.argmax()), 5, 7, 11]
    keep = [[t.clone() for t in (m.S, m.conv, m.kc, m.vc)] for m in tp]

    def restore(r):
        for t, k in zip((tp[r].S, tp[r].conv, tp[r].kc, tp[r].vc), keep[r]):
            t.copy_(k)

    verify = ranks.run(lambda r: tp[r].verify(0, toks, 90, ckpt_base=3)[0].clone())
    assert torch.equal(verify[0], verify[1])
    for t in range(4):
        if t == 0:
            ranks.run(restore)
        one = ranks.run(lambda r: tp[r].decode([toks[t]], [90 + t], [0])[0].clone())
        assert torch.equal(one[0], one[1]) and torch.equal(one[0][0], verify[0][t]), t
        assert _rel(one[0], ref.decode([toks[t]], [90 + t], [0])[0]) < NOISE
    ranks.run(restore)
    pair = ranks.run(lambda r: tp[r].decode([toks[0], 9], [90, 0], [0, 1])[0].clone())
    assert torch.equal(pair[0][0], verify[0][0])
    torch.cuda.synchronize()
    lib.check_err_word()


def test_two_ranks_moe():
    """Expert-parallel model with int8 mixers and a sharded int8 shared expert, the reference's router logits lent to it."""
    from velogb10_b200.models.runtime import GpuModel
    from velogb10_b200.ops import lib
    cfg, ranks = _cfg(True), _Ranks(2)
    ref = GpuModel(_as_bf16(_weights(cfg)), keep_canonical=True)
    tp = [GpuModel(_weights(cfg, r, 2), comm=ranks.comms[r]) for r in range(2)]
    assert all(any(q.fmt == "int8" for n, q in m.w.linears() if "shared" in n) for m in tp)
    for m in [ref] + tp:
        m.alloc_state(2, 2 + 17, 256)
    seen = []
    ref.router_logits_hook = lambda lg, n: seen.append(lg[:n].clone())
    prompt = torch.randint(0, cfg.vocab_size, (60,), generator=torch.Generator().manual_seed(5)).tolist()

    def lent(r, run):
        it = iter(seen)
        tp[r].router_logits_hook = lambda lg, n: lg[:n].copy_(next(it))
        return run(tp[r]).clone()

    for run in (lambda m: m.prefill(0, prompt)[0], lambda m: m.decode([5], [60], [0])[0], lambda m: m.decode([7, 9], [61, 0], [0, 1])[0]):
        seen.clear()
        want = run(ref).clone()
        got = ranks.run(lambda r: lent(r, run))
        assert torch.equal(got[0], got[1]) and _rel(got[0], want) < NOISE, _rel(got[0], want)
    torch.cuda.synchronize()
    lib.check_err_word()
