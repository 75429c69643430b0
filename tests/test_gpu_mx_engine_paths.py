"""Engines with a block-scaled full-context cache: the rows that a SnapKV draft keeps, sequences of unequal lengths that come and go, speculation of two
models, tensor-parallel shards."""
import os
import subprocess
import sys
import tempfile
from pathlib import Path

import pytest
import torch

from tests import golden_cfg as gc
from tests import mx_util as mx

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF = torch.bfloat16
KINDS = ["mxfp8", "mxfp4"]
# how far logits may be off those over a 16-bit cache, relative, in 2-norms: as much as an element of the cache is off at most
OFF = {"mxfp8": 2.0 ** -4, "mxfp4": 0.25}


def checkpoints(**models):
    """A folder of checkpoints, name = (config, weights)."""
    from magicdec_amd.Engine import model_core
    d = tempfile.mkdtemp(prefix="md_mx_ckpt_")
    for name, (cfg, sd) in models.items():
        os.makedirs(os.path.join(d, name))
        torch.save(sd, os.path.join(d, name, "model.pth"))
        model_core.transformer_configs[name] = gc.config_kwargs(cfg)
    return Path(d)


@pytest.fixture(scope="module")
def ckpt():
    return checkpoints(**{name: gc.tiny(name) for name in gc.TINY})


@pytest.fixture(scope="module")
def ids():
    return gc.synthetic_batches()[0].to(DEV)


def target(path, kv_dtype, graphs=False, batch=gc.B, **more):
    from magicdec_amd.Engine.SnapKV.backend import LMBackend
    eng = LMBackend(dtype=BF, device=DEV, dec_len=gc.GAMMA + 1, **(dict(draft_dec_len=1) if "draft_budget" in more else {}))
    eng.load_model(path / "model.pth", use_tp=False)
    if graphs:
        eng.compile()
    eng.setup_caches(max_batch_size=batch, max_seq_length=gc.MAX_LEN, kv_dtype=kv_dtype, **more)
    return eng


def off(a, b):
    return ((a.float() - b.float()).norm() / b.float().norm()).item()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("name", ["tinytgt", "tinyqwen"])
def test_the_snapkv_draft_keeps_the_rows_of_a_select_over_the_same_values(ckpt, ids, kind, name, monkeypatch):
    """In every layer the draft cache is, bit for bit, what the select makes of a 16-bit cache that holds the block-scaled one's values (which bf16 holds
    exactly), with the same queries."""
    from magicdec_amd import ops
    from magicdec_amd.Engine import model_core
    eng = target(ckpt / name, kind, draft_budget=gc.BUDGET)
    calls = []
    select = model_core.Transformer._select_mx

    def recorded(self, q_rot, cache, tab, draft_cache, snap_tab):
        before = (q_rot.clone(), cache.clone(), [t.clone() for t in (tab.indices, tab.indptr, tab.last_page_len)], draft_cache.clone(),
                  [t.clone() for t in (snap_tab.indices, snap_tab.indptr, snap_tab.last_page_len)], self._snap_ctx_len)
        select(self, q_rot, cache, tab, draft_cache, snap_tab)
        calls.append((*before, draft_cache.clone()))
    monkeypatch.setattr(model_core.Transformer, "_select_mx", recorded)
    eng.encode(ids)
    assert len(calls) == len(eng.model.layers)
    D = calls[0][0].shape[-1]
    for q_rot, cache, (indices, indptr, last), draft, snap, ctx, got in calls:
        assert ctx == ids.shape[1]
        values = mx.dequantize(*mx.unpack(cache.cpu(), kind, D), kind)
        plain = values.to(BF)
        assert torch.equal(plain.double(), values)
        ops.snapkv_select(q_rot, plain.to(DEV), indices, indptr, ctx, eng.model.window_size, gc.BUDGET, model_core.POOL_KERNEL, draft, *snap,
                          ops.AttnWorkspace(DEV), kv_layout="HND")
        assert torch.equal(draft.view(torch.int16), got.view(torch.int16))
        # the draft's rows are among the request's, none twice (rows of random weights are all different)
        per = got.shape[0] // gc.B
        for b in range(gc.B):
            rows = got[b * per:(b + 1) * per, 0].reshape(-1, *got.shape[3:])[:gc.BUDGET].flatten(1)
            assert rows.unique(dim=0).shape[0] == gc.BUDGET


@pytest.mark.parametrize("kind", KINDS)
def test_sequences_of_unequal_lengths(ckpt, kind):
    """step(): a prompt's portion beside a single token, a sequence that ends, one that takes its pages, against the same of a 16-bit cache.  The first layer's
    rows are the 16-bit engine's, quantised."""
    g = torch.Generator().manual_seed(7)
    text = {s: torch.randint(4, 2048, (n,), generator=g) for s, n in (("a", 330), ("b", 90), ("c", 140), ("d", 260))}
    logits, rows = {}, {}
    for kv in ("bf16", kind):
        eng = target(ckpt / "tinytgt", kv, batch=3)
        got = []

        def step(*parts):
            entries = [(s, text[s][a:b]) for s, a, b in parts]
            _, lg = eng.step(entries, want=[[len(t) - 1] for _, t in entries])
            got.append(lg.float().cpu())
        step(("a", 0, 300), ("b", 0, 77))
        step(("a", 300, 301), ("c", 0, 130), ("b", 77, 78))
        eng.end("b")
        step(("d", 0, 250), ("a", 301, 305), ("c", 130, 131))
        step(("a", 305, 306), ("c", 131, 132), ("d", 250, 251))
        cache = eng.model.layers[0].attention.kv_cache.kv_cache.cpu()
        logits[kv], rows[kv] = got, {}
        for s, (_, pages, n) in eng.pool.seqs.items():
            if kv == "bf16":
                mine = mx.quantize(cache[pages], kind)
            else:
                code, scale = mx.unpack(cache, kind, 64)
                mine = code[pages], scale[pages]
            rows[kv][s] = [x.permute(1, 2, 0, 3, 4).flatten(2, 3)[:, :, :n] for x in mine]
        assert sorted(rows[kv]) == ["a", "c", "d"]
    for s in rows["bf16"]:
        for a, b in zip(rows[kind][s], rows["bf16"][s]):
            assert torch.equal(a, b), s
    for a, b in zip(logits[kind], logits["bf16"]):
        assert off(a, b) <= OFF[kind]
        assert not torch.equal(a, b)


def test_speculation_of_two_models(ids):
    """A target with a block-scaled cache and a SnapKV draft model, whose next tokens stand far above the others: the tokens of a 16-bit cache's run, with
    captured steps and without."""
    from magicdec_amd import harness
    from magicdec_amd.Engine.SnapKV.backend_draft import LMBackend_Draft
    (cfg_t, sd_t), (cfg_d, sd_d) = gc.peaked_pair()
    d = checkpoints(peakedtgt=(cfg_t, sd_t), peakeddrf=(cfg_d, sd_d))
    runs = {}
    for kv, graphs in (("bf16", False), ("mxfp8", False), ("mxfp8", True), ("mxfp4", False), ("mxfp4", True)):
        tgt = target(d / "peakedtgt", kv, graphs)
        drf = LMBackend_Draft(dtype=BF, device=DEV, draft_budget=gc.BUDGET)
        drf.load_model(d / "peakeddrf" / "model.pth", use_tp=False)
        if graphs:
            drf.compile()
        drf.setup_caches(max_batch_size=gc.B, max_seq_length=gc.MAX_LEN, draft_budget=gc.BUDGET)
        st, _ = harness.run_longspec_batch(tgt, drf, ids, gc.GAMMA, gc.MAX_LEN, gc.EOT_1, gc.EOT_2)
        assert st.iters > 3
        runs[kv, graphs] = st.output.cpu(), st.num_nodes.cpu(), tgt.cachelens.cpu()
    for run in runs.values():
        for a, b in zip(run, runs["bf16", False]):
            assert torch.equal(a, b)


@pytest.mark.parametrize("kind", KINDS)
def test_tensor_parallel_shards(ckpt, ids, kind):
    """Two ranks on one GPU, a kv head each: their caches' first layer is the whole engine's, head by head, but for elements on the edge of their roundings;
    logits are as far off the whole engine's as the cache's elements are at most; both ranks end with the same tokens."""
    out = tempfile.mkdtemp(prefix="md_mx_tp_")
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    port = 29900 + os.getpid() % 90 + KINDS.index(kind)
    procs = []
    for r in range(2):
        env = dict(os.environ, LOCAL_RANK=str(r), LOCAL_WORLD_SIZE="2", RANK=str(r), WORLD_SIZE="2", MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port),
                   MD_CKPT=str(ckpt), MD_OUT=out, MD_KV_DTYPE=kind, MAGICDEC_TP_SINGLE_GPU="1", MAGICDEC_ONESHOT_AR="1", HSA_ENABLE_IPC_MODE_LEGACY="0")
        procs.append(subprocess.Popen([sys.executable, os.path.join(root, "tests", "_tp_mx_worker.py")], env=env, stdout=subprocess.PIPE,
                                      stderr=subprocess.STDOUT, text=True))
    logs = []
    try:
        for p in procs:
            logs.append(p.communicate(timeout=100)[0])
    finally:
        for p in procs:
            if p.poll() is None:
                p.kill()
    assert all(p.returncode == 0 for p in procs), "\n".join(log[-3000:] for log in logs)
    ranks = [torch.load(os.path.join(out, f"rank{r}.pt")) for r in range(2)]
    assert torch.equal(ranks[0]["output"], ranks[1]["output"]) and torch.equal(ranks[0]["num_nodes"], ranks[1]["num_nodes"])
    assert ranks[0]["iters"] == ranks[1]["iters"] > 3
    eng = target(ckpt / "tinytgt", kind)
    eng.encode(ids)
    whole = mx.unpack(eng.model.layers[0].attention.kv_cache.kv_cache.cpu(), kind, 64)
    for r in range(2):
        code, scale = mx.unpack(ranks[r]["cache"], kind, 64)
        assert code.shape[2] == 1
        differ = (mx.dequantize(code, scale, kind) != mx.dequantize(whole[0][:, :, r:r + 1], whole[1][:, :, r:r + 1], kind)).float().mean().item()
        assert differ <= 0.02
    eng.inference(ids[:, :gc.GAMMA + 1].clone())
    assert off(torch.cat([rank["logits"] for rank in ranks], 1), eng.model._last_logits.cpu()) <= OFF[kind]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("name,streaming", [("tiny70b", False), ("tinyqwen", False), ("tinytgt", True), ("tiny70b", True)])
def test_self_speculation_of_other_models(ckpt, ids, kind, name, streaming):
    """Eight query heads of 128 on a kv head, five of 64, and the StreamingLLM draft beside a block-scaled verify cache: a verify step's logits near those over
    16-bit pages, and a whole run with captured steps the run without, token for token."""
    from magicdec_amd import harness
    from magicdec_amd.Engine.StreamingLLM.backend import LMBackend as Streaming
    logits, runs = {}, []
    for kv, graphs in (("bf16", False), (kind, False), (kind, True)):
        if streaming:
            eng = Streaming(dtype=BF, device=DEV, dec_len=gc.GAMMA + 1)
            eng.load_model(ckpt / name / "model.pth", use_tp=False)
            if graphs:
                eng.compile()
            eng.setup_caches(max_batch_size=gc.B, max_seq_length=gc.MAX_LEN, draft_budget=gc.BUDGET, kv_dtype=kv)
        else:
            eng = target(ckpt / name, kv, graphs, draft_budget=gc.BUDGET)
        eng.encode(ids)
        eng.verify(ids[:, :gc.GAMMA + 1].clone())
        logits[kv] = eng.model._last_logits.float().cpu()
        st, _ = harness.run_selfspec_batch(eng, ids, gc.GAMMA, gc.MAX_LEN, gc.EOT_1, gc.EOT_2, streaming)
        assert st.iters > 3 and bool((st.num_nodes.cpu() > ids.shape[1]).all())
        if kv == kind:
            runs.append((st.output.cpu(), st.num_nodes.cpu(), eng.cachelens.cpu()))
    assert 0 < off(logits[kind], logits["bf16"]) <= OFF[kind]
    for a, b in zip(*runs):
        assert torch.equal(a, b)
